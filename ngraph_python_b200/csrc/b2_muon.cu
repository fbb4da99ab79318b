// One optimizer step over many matrices whose updates are orthogonalised:
//
//   mean = mu mean + (1 - mu) g,  u = (1 - mu) g + mu mean,  x = u / (|u| + eps)
//   `steps` times:  A = x x^T,  B = a I + b A + c A A,  x = B x          (x^T x and x B where there are more rows than columns)
//   param = param (1 - lr wd decay) - lr scale x
//
// Bound by the tensor cores: 3 n^2 m + n^3 operations a step for n x m (of both squares, which are symmetric, half), three times
// over, for what comes near fp32.  x, A and B are held as two fp16 parts, hi = the value rounded to fp16, lo = the rest rounded to
// fp16: together off by up to 2^-23 of the value, where fp32 rounds to 2^-24; of (hi + lo)(hi' + lo') the product lo lo' is
// left out, up to 2^-22 of the whole.  fp16 has the range for it because the largest singular value of every operand is
// known beforehand: x is normalised, and what the polynomial makes of [0, s] is worked out on the host, which gives each operand
// a power of two that puts its largest possible value next to the largest of fp16.  Values down to 2^-18 of it keep all of
// their lo part, those below 2^-29 none: it ends at fp16's last bit, 2^-41 of the largest.  So the update is as exact as one of fp32
// products in the norm of the matrix (640 x 1920: 2.8e-6 of it, numpy's fp32 2.2e-6), but rows a million times smaller than others are
// off by 4e-5 of themselves, where fp32 has 3e-7.
// (Three tf32 products give the same accuracy at half the rate; bf16 parts have 8 bits each, 2^-17 together.)
//
// Storage: blocks of 64 x 64 values, hi and lo behind one another, each 8 KB as the tensor core reads it from shared memory
// (rows of 128 bytes whose 16-byte pieces are swizzled by the row), so that an operand tile is a few bulk copies without a
// descriptor, whatever the matrix's own rows are like.  A block serves as rows of an operand (its k along the columns) and
// as columns of one (k along the rows) alike: the instruction reads both, so that x is neither transposed nor kept twice.
// What lies outside the matrix is zero and stays zero.
//
// Three launches for all matrices and steps: the mean and the sums of squares; x in parts; the products (a fourth for small
// matrices).  The products are
// one launch for all steps: work items -- a tile of A, B or x of one matrix -- are numbered so that what an item reads has lower
// numbers, CTAs take the next number when they are done with one, and an item waits until its matrix has counted the items
// that it reads.  Only items that a running CTA has taken are waited for, so that it does not matter how many CTAs run.
// With a launch for each product the last wave of tiles of every one of 15 would leave SMs idle.
//
// 48 matrices of 12 layers of 640 (59 million values): 2.95 ms in a loop, where power caps the clock, 2.5 alone; the 16-bit products
// by themselves would take 1.14 at the rate of a large product, 1.35 at its sustained one.  A tile of 256 columns keeps shared memory busy for
// 1920 of the 1960 cycles of a block of k (144 KB read by the tensor core, 96 KB written by the copies, 128 bytes a cycle); what comes
// on top is the storing of tiles, some 5000 cycles after ten blocks of k, which the next tile's first two blocks hide in part.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <new>
#include <vector>

#include <cuda_fp16.h>

#include "b2_gemm_impl.cuh"
#include "b2_operators.h"

namespace {

constexpr int kMeanThreads = 256;
constexpr int kMostSteps = 32;
constexpr long long kMostSide = 1 << 20, kMostShort = 1 << 15;
constexpr int kBlock = 64;                                  // rows and columns of a block
constexpr int kBlockBytes = kBlock * kBlock * 2;            // of one part
constexpr int kBlockPair = 2 * kBlockBytes;

enum { GRAM = 0, POLY = 1, MULTIPLY = 2 };

// One matrix.  Offsets are bytes of the scratch, from the first plane on.
struct Matrix {
    float* param;
    const float* grad;
    float* mean;
    long long x[2], square, poly, held;      // two turns of x [row blocks][column blocks], A and B [n blocks][n blocks], A in fp32
    int rows, cols, row_blocks, col_blocks, n_blocks, tall;
    int items[3];                            // of a step, by phase
    int first_chunk, chunks;
    float decay, scale;
};
struct Chunk {                               // values of a matrix whose squares one CTA adds
    int matrix, n;
    long long at;
};
struct Block {                               // one block of x
    int matrix, at;
};
struct Item {                                // a tile: 128 rows from block 2 i on, `width` blocks of columns from block j on
    int matrix;
    short phase, width;
    int i, j;
};
struct Group {                               // matrices whose steps run next to one another; items of one step
    long long first, count;
};
struct Header {
    long long matrices, chunks, items, blocks, solos, bytes, groups;      // bytes: of the scratch
};
constexpr size_t kHeader = 64;

struct Layout {
    std::vector<Matrix> matrices;
    std::vector<Chunk> chunks;
    std::vector<Block> blocks;
    std::vector<Item> items;
    std::vector<Group> groups;
    long long solos;                         // the last of the matrices, which have a CTA to themselves
    long long bytes;                         // of planes
    size_t plan_bytes() const {
        return kHeader + matrices.size() * sizeof(Matrix) + chunks.size() * sizeof(Chunk) + blocks.size() * sizeof(Block) + items.size() * sizeof(Item) +
               groups.size() * sizeof(Group);
    }
};

struct Rates {
    float mu, rest, eps;
    double lr, wd;
    int nesterov;
};
// Powers of two that operands are stored with, by step, and the polynomial.
struct Poly {
    float a, b, c;
    int steps;
    signed char x[kMostSteps + 1], square[kMostSteps], poly[kMostSteps];
};
__device__ __forceinline__ float power(int e) { return __int_as_float((e + 127) << 23); }

__device__ __forceinline__ const Header* header_of(const void* plan) { return static_cast<const Header*>(plan); }
__device__ __forceinline__ const Matrix* matrices_of(const void* plan) { return reinterpret_cast<const Matrix*>(static_cast<const char*>(plan) + kHeader); }
__device__ __forceinline__ const Chunk* chunks_of(const void* plan) { return reinterpret_cast<const Chunk*>(matrices_of(plan) + header_of(plan)->matrices); }
__device__ __forceinline__ const Block* blocks_of(const void* plan) { return reinterpret_cast<const Block*>(chunks_of(plan) + header_of(plan)->chunks); }
__device__ __forceinline__ const Item* items_of(const void* plan) { return reinterpret_cast<const Item*>(blocks_of(plan) + header_of(plan)->blocks); }
__device__ __forceinline__ const Group* groups_of(const void* plan) { return reinterpret_cast<const Group*>(items_of(plan) + header_of(plan)->items); }

struct Told {                                // what the caller says of the plan; a step with other sizes does nothing
    long long matrices, chunks, items, blocks, solos, bytes;
};
__device__ __forceinline__ bool fits(const void* plan, const Told& t) {
    const Header* h = header_of(plan);
    return h->matrices == t.matrices && h->chunks == t.chunks && h->items == t.items && h->blocks == t.blocks && h->solos == t.solos &&
           h->bytes == t.bytes;
}

// The scratch: sums of squares by chunk; counters; planes.
struct Room {
    double* sums;
    unsigned* next;                          // the number of the next item, whether a wait ran out, and by matrix the items done
    unsigned* failed;
    unsigned* done;
    char* planes;
};

template <int THREADS>
__device__ __forceinline__ double cta_sum(double q, double* words) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) words[threadIdx.x >> 5] = q;
    __syncthreads();
    q = 0.0;
    for (int w = 0; w < THREADS / 32; ++w) q += words[w];
    return q;
}

// The mean of a chunk and the sum of squares of its u, in 64 bits: squares of any gradient fit.  Memory bounds it: 59 million values in
// 104 us, 12 bytes each at 6.8 TB/s (168 us with loads of one value).
__global__ void __launch_bounds__(kMeanThreads, 4)
muon_mean_kernel(const void* plan, const Told told, const Rates r, const float* grad_scale, float* step, const Room room) {
    __shared__ double words[kMeanThreads / 32];
    after_earlier_kernels();
    if (!fits(plan, told)) return;
    if (blockIdx.x == 0) {
        if (threadIdx.x == 0 && step) *step += 1.0f;
        if (threadIdx.x == 0) *room.next = *room.failed = 0;
        for (long long i = threadIdx.x; i < told.matrices; i += kMeanThreads) room.done[i] = 0;
    }
    const float s = grad_scale ? *grad_scale : 1.0f;
    for (long long k = blockIdx.x; k < told.chunks; k += gridDim.x) {
        const Chunk c = chunks_of(plan)[k];
        const Matrix& t = matrices_of(plan)[c.matrix];
        const float* grad = t.grad + c.at;
        float* mean = t.mean + c.at;
        double q = 0.0;
        const auto next = [&](float g, float& m) {
            m = r.mu * m + r.rest * (g * s);
            const float u = r.nesterov ? r.rest * (g * s) + r.mu * m : m;
            q = fma((double)u, (double)u, q);
        };
        // by fours where the tensors lie so, all of a thread's loads before the first is used
        constexpr int AHEAD = 4;
        const int whole = (((uintptr_t)grad | (uintptr_t)mean) & 15) == 0 ? c.n / 4 : 0;
        for (int i0 = threadIdx.x; i0 < whole; i0 += AHEAD * kMeanThreads) {
            float4 g[AHEAD], m[AHEAD];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
                if (i0 + j * kMeanThreads < whole) {
                    g[j] = reinterpret_cast<const float4*>(grad)[i0 + j * kMeanThreads];
                    m[j] = reinterpret_cast<const float4*>(mean)[i0 + j * kMeanThreads];
                }
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
                if (i0 + j * kMeanThreads < whole) {
                    next(g[j].x, m[j].x);
                    next(g[j].y, m[j].y);
                    next(g[j].z, m[j].z);
                    next(g[j].w, m[j].w);
                    reinterpret_cast<float4*>(mean)[i0 + j * kMeanThreads] = m[j];
                }
        }
        for (int i0 = 4 * whole + threadIdx.x; i0 < c.n; i0 += 2 * AHEAD * kMeanThreads) {
            float g[2 * AHEAD], m[2 * AHEAD];
#pragma unroll
            for (int j = 0; j < 2 * AHEAD; ++j)
                if (i0 + j * kMeanThreads < c.n) {
                    g[j] = grad[i0 + j * kMeanThreads];
                    m[j] = mean[i0 + j * kMeanThreads];
                }
#pragma unroll
            for (int j = 0; j < 2 * AHEAD; ++j)
                if (i0 + j * kMeanThreads < c.n) {
                    next(g[j], m[j]);
                    mean[i0 + j * kMeanThreads] = m[j];
                }
        }
        q = cta_sum<kMeanThreads>(q, words);
        if (threadIdx.x == 0) room.sums[k] = q;
    }
}

// What u is multiplied by, one factor behind the other, for u * up / norm.  A norm of fp32 values may be more or less than fp32 holds,
// and so may its reciprocal: the first factor takes u by a power of two to where neither is.
__device__ __forceinline__ float2 over_norm(double norm, float up) {
    const int e = ((__double2hiint(norm) >> 20) & 0x7ff) - 1023;
    const int first = e > 100 ? -100 : e < -100 ? 100 : 0;
    return make_float2(power(first), (float)((double)up * (double)power(-first) / norm));
}

// Two values as two fp16 parts each
__device__ __forceinline__ void parts(float u, float v, unsigned& hi, unsigned& lo) {
    const __half2 h = __floats2half2_rn(u, v);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(u - f.x, v - f.y);
    hi = *reinterpret_cast<const unsigned*>(&h);
    lo = *reinterpret_cast<const unsigned*>(&l);
}
// Eight values next to one another of row `row` of a block, 8 `piece` columns in
__device__ __forceinline__ void put_piece(char* block, int row, int piece, const float* v, int to_lo = kBlockBytes) {
    uint4 hi, lo;
    parts(v[0], v[1], hi.x, lo.x);
    parts(v[2], v[3], hi.y, lo.y);
    parts(v[4], v[5], hi.z, lo.z);
    parts(v[6], v[7], hi.w, lo.w);
    char* at = block + row * 128 + ((piece ^ (row & 7)) << 4);
    *reinterpret_cast<uint4*>(at) = hi;
    *reinterpret_cast<uint4*>(at + to_lo) = lo;
}
// x of the first step, a block at a time.  A CTA's blocks lie next to one another, so that it adds a matrix's sums of squares once.
// 59 million values in 109 us (249 with loads of one value and the sums added for every block).
__global__ void __launch_bounds__(kMeanThreads, 4)
muon_parts_kernel(const void* plan, const Told told, const Rates r, const float* grad_scale, int exponent, const Room room) {
    __shared__ double words[kMeanThreads / 32];
    after_earlier_kernels();
    if (!fits(plan, told)) return;
    const float s = grad_scale ? *grad_scale : 1.0f;
    const long long run = (told.blocks + gridDim.x - 1) / gridDim.x, end = min((blockIdx.x + 1) * run, told.blocks);
    float2 factors = make_float2(0.0f, 0.0f);
    int matrix = -1;
    for (long long k = blockIdx.x * run; k < end; ++k) {
        const Block c = blocks_of(plan)[k];
        const Matrix& t = matrices_of(plan)[c.matrix];
        if (c.matrix != matrix) {
            double q = 0.0;
            for (int i = threadIdx.x; i < t.chunks; i += kMeanThreads) q += room.sums[t.first_chunk + i];
            factors = over_norm(sqrt(cta_sum<kMeanThreads>(q, words)) + (double)r.eps, power(exponent));
            matrix = c.matrix;
        }
        const int rb = c.at / t.col_blocks, cb = c.at - rb * t.col_blocks;
        char* block = room.planes + t.x[0] + (long long)c.at * kBlockPair;
        // a thread's two runs of eight values, by fours where the tensors' rows lie so
        constexpr int EACH = kBlock * 8 / kMeanThreads;
        const bool vec = (((uintptr_t)t.grad | (uintptr_t)t.mean) & 15) == 0 && (t.cols & 3) == 0;
        const int piece = threadIdx.x & 7, at_col = cb * kBlock + piece * 8;
        float g[EACH][8], m[EACH][8];
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const int at_row = rb * kBlock + (threadIdx.x >> 3) + e * (kMeanThreads / 8);
            const long long at = (long long)at_row * t.cols + at_col;
            const int there = at_row < t.rows ? t.cols - at_col : 0;
            if (vec) {
#pragma unroll
                for (int j = 0; j < 8; j += 4) {
                    float4 a = make_float4(0, 0, 0, 0), b = a;
                    if (j < there) {
                        a = *reinterpret_cast<const float4*>(t.mean + at + j);
                        if (r.nesterov) b = *reinterpret_cast<const float4*>(t.grad + at + j);
                    }
                    m[e][j] = a.x; m[e][j + 1] = a.y; m[e][j + 2] = a.z; m[e][j + 3] = a.w;
                    g[e][j] = b.x; g[e][j + 1] = b.y; g[e][j + 2] = b.z; g[e][j + 3] = b.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    m[e][j] = j < there ? t.mean[at + j] : 0.0f;
                    g[e][j] = j < there && r.nesterov ? t.grad[at + j] : 0.0f;
                }
            }
        }
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float u = r.nesterov ? r.rest * (g[e][j] * s) + r.mu * m[e][j] : m[e][j];
                m[e][j] = u * factors.x * factors.y;
            }
            // (what lies outside the matrix is zero, whatever the factors are)
            const int at_row = rb * kBlock + (threadIdx.x >> 3) + e * (kMeanThreads / 8), there = at_row < t.rows ? t.cols - at_col : 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) m[e][j] = j < there ? m[e][j] : 0.0f;
            put_piece(block, (threadIdx.x >> 3) + e * (kMeanThreads / 8), piece, m[e]);
        }
    }
}

// ---- the products ------------------------------------------------------------------------------------------
constexpr int kUnit = 32 << 10, kUnits = 5;                 // the ring: both parts of 128 rows of P, of Q up to 128, or one part of more
constexpr int kQueue = 4;
constexpr int kEpilogueWarps = 8;
constexpr int kProductThreads = 128 + 32 * kEpilogueWarps;  // (a warp group for the two that copy and multiply)
// Registers of a thread: 168 at the start, of which the first group gives so many to the epilogue's two, 56 + 2 x 224 = 3 x 168
constexpr int kFewRegisters = 56, kManyRegisters = 224;
static_assert(kFewRegisters + 2 * kManyRegisters <= 3 * 168, "what the block was launched with");
constexpr int kPairs = kEpilogueWarps / 2;                  // two warps of the epilogue have the rows of a block
constexpr int kRooms = 2 * kPairs;                          // for a part of a block each
constexpr int kProductShared = 1024 + kUnits * kUnit + kRooms * kBlockBytes + 512;
static_assert(kProductShared <= 227 << 10, "shared memory of a CTA");
// Blocks of k that are added in tensor memory, whose sums lose what they add: 640 x 1920 is 2.8e-6 off in the 2-norm with one
// (numpy's fp32 2.2e-6), 6.4e-6 with two, 1.2e-5 with four, for 2.97, 2.82 and 2.73 ms of 48 matrices.  The small products
// go first.  The rest is added in registers.
constexpr int kChain = 1;
constexpr int kDependencyPolls = 1 << 22;

struct Work {
    int matrix, phase, step, i, j, width, k_blocks;
};
// Where the blocks of an operand lie: 128 rows (or columns) of tiles by `mn`, k by `k`, in blocks
struct Operand {
    const char* base;
    int mn, k, last;
    unsigned major;                          // 1: k along the rows of the storage
};
__device__ __forceinline__ Operand operand_of(const Matrix& t, const char* planes, int phase, int turn, bool second) {
    const bool x = phase == GRAM || (phase == MULTIPLY && (second != (t.tall != 0)));
    if (!x) return {planes + (phase == POLY ? t.square : t.poly), t.n_blocks, 1, t.n_blocks - 1, 0};
    const char* base = planes + t.x[turn];
    const bool columns = phase == GRAM ? t.tall != 0 : second;
    if (columns) return {base, 1, t.col_blocks, t.col_blocks - 1, 1};
    return {base, t.col_blocks, 1, t.row_blocks - 1, 0};
}
// a shared-memory descriptor: 128-byte swizzle, groups of eight rows 1024 bytes apart; k along the rows: groups of 64 columns a block apart
__device__ __forceinline__ unsigned long long describe(unsigned address, unsigned major) {
    unsigned long long d = (address >> 4) & 0x3FFF;
    d |= (unsigned long long)(major ? kBlockBytes >> 4 : 1) << 16;
    d |= (unsigned long long)(1024 >> 4) << 32;
    d |= (unsigned long long)1 << 46;
    d |= (unsigned long long)2 << 61;
    return d;
}
__device__ __forceinline__ void multiply_f16(unsigned d, unsigned long long a, unsigned long long b, unsigned instruction, unsigned accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(instruction), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void copy_block(unsigned to, const char* from, unsigned bytes, unsigned long long* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(to), "l"(from), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ unsigned load_acquire(const unsigned* p) {
    unsigned v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}

__device__ __forceinline__ bool test_wait(unsigned long long* bar, unsigned parity) {       // without waiting
    unsigned ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}

__global__ void __launch_bounds__(kProductThreads, 1)
muon_product_kernel(const void* plan, const Told told, const Rates r, const Poly poly, const float* lr, const Room room, int* status) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    char* rooms = reinterpret_cast<char*>(smem + kUnits * kUnit);
    unsigned long long* full_bar = reinterpret_cast<unsigned long long*>(smem + kUnits * kUnit + kRooms * kBlockBytes);
    unsigned long long* empty_bar = full_bar + kUnits;
    unsigned long long* sum_full = empty_bar + kUnits;          // [2]
    unsigned long long* sum_empty = sum_full + 2;               // [2]
    unsigned long long* queue_full = sum_empty + 2;
    unsigned long long* queue_empty = queue_full + kQueue;
    unsigned long long* idle = queue_empty + kQueue;
    Work* queue = reinterpret_cast<Work*>(idle + 1);
    unsigned* tmem_holder = reinterpret_cast<unsigned*>(queue + kQueue);
    int* fail_flag = reinterpret_cast<int*>(tmem_holder + 1);

    const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kUnits; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(&sum_full[b], 1); mbar_init(&sum_empty[b], kEpilogueWarps); }
        for (int q = 0; q < kQueue; ++q) { mbar_init(&queue_full[q], 1); mbar_init(&queue_empty[q], 1 + kEpilogueWarps); }
        mbar_init(idle, 1);
        *fail_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(tmem_holder, 512);
    // (the launch for small matrices goes by this: where it starts, all that came before this kernel has ended)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem_base = (unsigned)warp_uniform((int)*tmem_holder);
    const bool mine = fits(plan, told);                         // (else no item is taken)
    const Matrix* matrices = matrices_of(plan);

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegisters));
        if (warp == 0) {
            // A lane to each copy of a block of k, with its addresses worked out once an item: one thread for all of them took 150 cycles a
            // copy, 1900 a block of k of 256 columns, of which the products take 1536.
            int s = 0, q = 0;
            unsigned parity = 1, queue_parity = 1;
            bool ok = true;
            long long group = 0, issued = 0;                    // units that copies have been started into
            const long long total = mine ? told.items * poly.steps : 0;
            for (;;) {
                // the next item
                Work w = {};
                w.phase = -1;
                long long number = total;
                if (lane == 0 && ok && total && !*reinterpret_cast<volatile unsigned*>(room.failed)) number = (long long)atomicAdd(room.next, 1u);
                number = __shfl_sync(0xffffffffu, number, 0);
                if (number < total) {
                    const Group* g = groups_of(plan) + group;
                    while (number >= poly.steps * (g->first + g->count)) { ++g; ++group; }
                    const long long in = number - poly.steps * g->first;
                    w.step = (int)(in / g->count);
                    const Item item = items_of(plan)[g->first + (in - w.step * g->count)];
                    const Matrix& t = matrices[item.matrix];
                    w.matrix = item.matrix;
                    w.phase = item.phase;
                    w.i = item.i;
                    w.j = item.j;
                    w.width = item.width;
                    w.k_blocks = item.phase == GRAM ? (t.tall ? t.row_blocks : t.col_blocks) : t.n_blocks;
                    // what it reads has been stored
                    const int before = w.step * (t.items[0] + t.items[1] + t.items[2]) + (item.phase > GRAM ? t.items[0] : 0) + (item.phase > POLY ? t.items[1] : 0);
                    const unsigned need = (unsigned)before * kEpilogueWarps;
                    bool there = false;
                    if (lane == 0)
                        for (int i = 0; i < kDependencyPolls && !there; ++i) {
                            there = (int)(load_acquire(room.done + item.matrix) - need) >= 0;
                            if (!there) {
                                if (*reinterpret_cast<volatile unsigned*>(room.failed)) break;
                                __nanosleep(40);
                            }
                        }
                    there = __shfl_sync(0xffffffffu, (int)there, 0) != 0;
                    asm volatile("fence.proxy.async;" ::: "memory");
                    if (!there) {
                        if (lane == 0) atomicExch(fail_flag, 1);
                        ok = false;
                        w.phase = -1;
                    }
                }
                if (!__all_sync(0xffffffffu, mbar_wait(&queue_empty[q], queue_parity))) {
                    if (lane == 0) atomicExch(fail_flag, 1);
                    ok = false;
                    break;
                }
                if (lane == 0) {
                    queue[q] = w;
                    mbar_arrive(&queue_full[q]);
                }
                if (++q == kQueue) { q = 0; queue_parity ^= 1u; }
                if (w.phase < 0) break;
                const Matrix& t = matrices[w.matrix];
                const Operand P = operand_of(t, room.planes, w.phase, w.step & 1, false), Q = operand_of(t, room.planes, w.phase, w.step & 1, true);
                // lanes 0 to 3: P, (part, block of rows); then Q, (part, block of columns), the lo part first.  Parts of Q in one unit up to 128
                // columns, behind it P; beyond, the lo part, P, the hi part: what is done with first makes room for what is wanted last
                const bool both = w.width <= 2, of_p = lane < 4;
                const int turn = of_p ? lane >> 1 : (lane - 4) / w.width, place = of_p ? lane & 1 : (lane - 4) % w.width;
                const int my_unit = of_p ? 1 : lane >= 4 + 2 * w.width ? -1 : both ? 0 : 2 * turn;
                const unsigned offset = (of_p ? turn * 2 + place : both ? turn * w.width + place : place) * kBlockBytes;
                const long long row = of_p ? (long long)min(2 * w.i + place, P.last) * P.mn : (long long)(w.j + place) * Q.mn;
                const char* from = (of_p ? P.base : Q.base) + row * kBlockPair + (of_p ? turn : turn ^ 1) * kBlockBytes;
                const long long along = (of_p ? P.k : Q.k) * (long long)kBlockPair;
                const int units = both ? 2 : 3;
                for (int kb = 0; kb < w.k_blocks && ok; ++kb) {
                    for (int u = 0; u < units; ++u) {
                        ok = __all_sync(0xffffffffu, mbar_wait(&empty_bar[s], parity));
                        if (!ok) {
                            if (lane == 0) atomicExch(fail_flag, 1);
                            break;
                        }
                        if (lane == 0) mbar_expect_tx(&full_bar[s], (u == 1 ? 4 : both ? 2 * w.width : w.width) * kBlockBytes);
                        __syncwarp();
                        if (my_unit == u) copy_block(smem_u32(smem + s * kUnit) + offset, from, kBlockBytes, &full_bar[s]);
                        ++issued;
                        if (++s == kUnits) { s = 0; parity ^= 1u; }
                    }
                    from += along;
                }
            }
            // copies in flight have landed before the CTA may end, whatever came of the others' waiting
            for (long long i = issued < kUnits ? 0 : issued - kUnits; i < issued; ++i)
                if (!__all_sync(0xffffffffu, mbar_wait(&full_bar[i % kUnits], (unsigned)(i / kUnits) & 1)) && lane == 0) atomicExch(fail_flag, 1);
        } else if (warp == 1) {
            if (elect_one()) {
                int s = 0, q = 0, chain = 0;
                unsigned parity = 0, queue_parity = 0;
                bool ok = true;
                auto wait_unit = [&] {
                    if (!mbar_wait(&full_bar[s], parity)) { atomicExch(fail_flag, 1); ok = false; }
                    tc_fence_after();
                    return smem_u32(smem + s * kUnit);
                };
                auto next = [&] { if (++s == kUnits) { s = 0; parity ^= 1u; } };
                while (ok) {
                    if (!mbar_wait_relaxed(&queue_full[q], queue_parity)) { atomicExch(fail_flag, 1); break; }
                    const Work w = queue[q];
                    mbar_arrive(&queue_empty[q]);
                    if (++q == kQueue) { q = 0; queue_parity ^= 1u; }
                    if (w.phase < 0) break;
                    const Matrix& t = matrices[w.matrix];
                    const unsigned p_major = operand_of(t, room.planes, w.phase, 0, false).major, q_major = operand_of(t, room.planes, w.phase, 0, true).major;
                    // fp16 operands, fp32 sums, 128 rows
                    const unsigned instruction = (1u << 4) | (p_major << 15) | (q_major << 16) | ((unsigned)(w.width * kBlock >> 3) << 17) | ((128u >> 4) << 24);
                    const unsigned p_step = p_major ? 2048 >> 4 : 32 >> 4, q_step = q_major ? 2048 >> 4 : 32 >> 4;       // 16 of k
                    const bool both = w.width <= 2;
                    for (int kb = 0; kb < w.k_blocks && ok; ++kb) {
                        const int in = kb % kChain, b = chain & 1;
                        if (in == 0) {
                            // the sums before in these columns have been read
                            if (chain > 1 && !mbar_wait(&sum_empty[b], ((chain >> 1) - 1) & 1)) { atomicExch(fail_flag, 1); ok = false; break; }
                            tc_fence_after();
                        }
                        const unsigned sum = tmem_base + b * 256;
                        const int q_unit = s;
                        unsigned q_at = wait_unit();
                        next();
                        const int p_unit = s;
                        const unsigned p_at = wait_unit();
                        next();
                        if (!ok) break;
                        const unsigned long long p_hi = describe(p_at, p_major), p_lo = describe(p_at + 2 * kBlockBytes, p_major);
                        unsigned long long q_part = describe(q_at, q_major);
#pragma unroll
                        for (int k = 0; k < 4; ++k) multiply_f16(sum, p_hi + k * p_step, q_part + k * q_step, instruction, in > 0 || k > 0);
                        int last_unit = q_unit;
                        if (both) {
                            q_part = describe(q_at + w.width * kBlockBytes, q_major);
                        } else {
                            tc_commit(&empty_bar[q_unit]);
                            last_unit = s;
                            q_at = wait_unit();
                            next();
                            if (!ok) break;
                            q_part = describe(q_at, q_major);
                        }
#pragma unroll
                        for (int k = 0; k < 4; ++k) multiply_f16(sum, p_lo + k * p_step, q_part + k * q_step, instruction, 1);
#pragma unroll
                        for (int k = 0; k < 4; ++k) multiply_f16(sum, p_hi + k * p_step, q_part + k * q_step, instruction, 1);
                        tc_commit(&empty_bar[p_unit]);
                        tc_commit(&empty_bar[last_unit]);
                        if (in == kChain - 1 || kb == w.k_blocks - 1) {
                            tc_commit(&sum_full[b]);
                            ++chain;
                        }
                    }
                }
                // products in flight have been made before tensor memory is freed
                tc_commit(idle);
                if (!mbar_wait(idle, 0)) atomicExch(fail_flag, 1);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegisters));
        // The epilogue: a quarter of the lanes (32 rows) to a warp, and every other block of columns.  Two warps have the rows of a block,
        // whose parts go to memory as whole blocks, by way of rooms in shared memory: stored from registers, sixteen bytes a row, a
        // tile of 256 columns took 13000 cycles, and 5000 more until the stores were done.
        const int quarter = warp & 3, half = (warp - 4) >> 2, in_row = (quarter & 1) * 32 + lane, pair = half * 2 + (quarter >> 1);
        const unsigned lanes = tmem_base + ((unsigned)(quarter * 32) << 16);
        char* space = rooms + pair * 2 * kBlockBytes;           // for both parts of a block
        const bool sender = (quarter & 1) == 0 && lane == 0;
        // The two warps meet as often as each other whatever becomes of their waits: of items both take the next one or neither, and where
        // sums did not come they store what they have, which is never said to be stored (of the param nothing).
        const auto together = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1 + pair) : "memory"); };
        const auto both_warps = [&](bool mine) {
            unsigned all;
            asm volatile(
                "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\t"
                "barrier.cta.red.and.pred q, %1, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                : "=r"(all) : "r"(1 + pair), "r"((unsigned)mine) : "memory");
            return all != 0;
        };
        int q = 0, chain = 0, stored = -1;                      // whose item has been sent, but is not said to be stored
        unsigned queue_parity = 0;
        bool ok = true;
        // An item is said to be stored when its copies have been made, which nobody waits for while there are other items: some blocks of k
        // into the next one.  (Waited for at once, 4000 cycles a tile.)
        const auto say = [&] {
            if (stored < 0) return;
            if (sender) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
            asm volatile("fence.proxy.async;" ::: "memory");
            __threadfence();
            __syncwarp();
            if (lane == 0) asm volatile("red.release.gpu.global.add.u32 [%0], %1;" ::"l"(room.done + stored), "r"(ok ? 1u : 0u) : "memory");
            stored = -1;
        };
        for (;;) {
            if (!__all_sync(0xffffffffu, test_wait(&queue_full[q], queue_parity))) say();
            if (!both_warps(mbar_wait_relaxed(&queue_full[q], queue_parity))) { atomicExch(fail_flag, 1); break; }
            const Work w = queue[q];
            __syncwarp();
            if (lane == 0) mbar_arrive(&queue_empty[q]);
            if (++q == kQueue) { q = 0; queue_parity ^= 1u; }
            if (w.phase < 0) break;
            if (w.phase == MULTIPLY && w.step == poly.steps - 1) {
                // the param's values are on their way into L2 meanwhile: a row to a lane, by 32 columns
                const Matrix& t = matrices[w.matrix];
                const int row = w.i * 128 + quarter * 32 + lane;
                for (int n = half; n < w.width; n += 2)
                    for (int c0 = 0; c0 < kBlock; c0 += 32) {
                        const int col = (w.j + n) * kBlock + c0;
                        if (row < t.rows && col < t.cols) asm volatile("prefetch.global.L2 [%0];" ::"l"(t.param + (long long)row * t.cols + col));
                    }
            }
            float sum[128];
#pragma unroll
            for (int j = 0; j < 128; ++j) sum[j] = 0.0f;
            for (int kb = 0; kb < w.k_blocks; kb += kChain, ++chain) {
                if (kb == 2 * kChain) say();
                const int b = chain & 1;
                if (ok && !__all_sync(0xffffffffu, mbar_wait(&sum_full[b], (chain >> 1) & 1))) { atomicExch(fail_flag, 1); ok = false; }
                tc_fence_after();
#pragma unroll
                for (int c0 = 0; c0 < 128; c0 += 32) {
                    const int n = half + 2 * (c0 >> 6);
                    if (n < w.width) {
                        unsigned v[32];
                        tmem_ld16(lanes + b * 256 + n * 64 + (c0 & 63), v);
                        tmem_ld16(lanes + b * 256 + n * 64 + (c0 & 63) + 16, v + 16);
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 32; ++j) sum[c0 + j] += __uint_as_float(v[j]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sum_empty[b]);
            }
            say();
            const Matrix& t = matrices[w.matrix];
            const int rb = 2 * w.i + (quarter >> 1), k = w.step;
            const bool last = w.phase == MULTIPLY && k == poly.steps - 1;
            const int row_blocks = w.phase == MULTIPLY ? t.row_blocks : t.n_blocks, col_blocks = w.phase == MULTIPLY ? t.col_blocks : t.n_blocks;
            char* planes = room.planes + (w.phase == GRAM ? t.square : w.phase == POLY ? t.poly : t.x[(k + 1) & 1]);
            const int into = w.phase == GRAM ? poly.square[k] - 2 * poly.x[k] : w.phase == POLY ? poly.poly[k] - 2 * poly.square[k] : poly.x[k + 1] - poly.x[k] - poly.poly[k];
            const float factor = w.phase == POLY ? poly.c * power(into) : last ? power(-poly.x[k] - poly.poly[k]) : power(into);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int n = half + 2 * i, cb = w.j + n;
                // of what is symmetric the upper half, stored twice
                if (n >= w.width || rb >= row_blocks || (w.phase != MULTIPLY && rb > cb)) continue;
                float* v = sum + 64 * i;
                if (w.phase == MULTIPLY) {
#pragma unroll
                    for (int j = 0; j < 64; ++j) v[j] *= factor;
                } else {
                    // A in fp32 for the step's second product, four values of a row and the next row's behind them
                    float4* held = reinterpret_cast<float4*>(room.planes + t.held + ((long long)rb * col_blocks + cb) * kBlockPair) + in_row;
                    const float linear = poly.b * power(poly.poly[k] - poly.square[k]), diagonal = poly.a * power(poly.poly[k]);
                    if (w.phase == GRAM) {
#pragma unroll
                        for (int j = 0; j < 64; ++j) v[j] *= factor;
#pragma unroll
                        for (int j = 0; j < 64; j += 4) __stcg(held + (j >> 2) * kBlock, make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]));
                    } else {
                        float4 old[16];                         // (all on their way before the first is used)
#pragma unroll
                        for (int j = 0; j < 16; ++j) old[j] = __ldcg(held + j * kBlock);
#pragma unroll
                        for (int j = 0; j < 64; ++j) {
                            const float4 four = old[j >> 2];
                            const float a = (j & 3) == 0 ? four.x : (j & 3) == 1 ? four.y : (j & 3) == 2 ? four.z : four.w;
                            v[j] = fmaf(linear, a, factor * v[j]);
                        }
                    }
                    if (w.phase == POLY && rb == cb && rb * kBlock + in_row < min(t.rows, t.cols)) {
#pragma unroll
                        for (int j = 0; j < 64; ++j)
                            if (j == in_row) v[j] += diagonal;
                    }
                }
                if (!last) {
                    // both parts, two values to a word, in the place of the values
                    unsigned hi[32], lo[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) parts(v[2 * j], v[2 * j + 1], hi[j], lo[j]);
                    const auto send = [&](char* to) {
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        together();
                        if (sender) {
                            // (both parts lie behind one another, here and there)
                            asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to), "r"(smem_u32(space)), "r"(kBlockPair) : "memory");
                            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                        }
                    };
                    const auto free_space = [&] {
                        if (sender) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                        together();
                    };
                    free_space();
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int at = in_row * 128 + ((e ^ (in_row & 7)) << 4);
                        *reinterpret_cast<uint4*>(space + at) = make_uint4(hi[4 * e], hi[4 * e + 1], hi[4 * e + 2], hi[4 * e + 3]);
                        *reinterpret_cast<uint4*>(space + kBlockBytes + at) = make_uint4(lo[4 * e], lo[4 * e + 1], lo[4 * e + 2], lo[4 * e + 3]);
                    }
                    send(planes + ((long long)rb * col_blocks + cb) * kBlockPair);
                    if (w.phase != MULTIPLY && rb < cb) {
                        // the block on the other side of the diagonal: 8 x 8 values at a time turned about on the way through registers, half
                        // of the rows to a warp
                        unsigned turned[2][8][4];
                        const unsigned base = smem_u32(space), mine = 4 * (quarter & 1) + (lane >> 3), in = lane & 7;
#pragma unroll
                        for (int part = 0; part < 2; ++part)
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                                             : "=r"(turned[part][e][0]), "=r"(turned[part][e][1]), "=r"(turned[part][e][2]), "=r"(turned[part][e][3])
                                             : "r"(base + part * kBlockBytes + (8 * mine + in) * 128 + ((e ^ in) << 4)) : "memory");
                        free_space();
#pragma unroll
                        for (int part = 0; part < 2; ++part)
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%4], {%0, %1, %2, %3};"
                                             ::"r"(turned[part][e][0]), "r"(turned[part][e][1]), "r"(turned[part][e][2]), "r"(turned[part][e][3]),
                                               "r"(base + part * kBlockBytes + (8 * e + in) * 128 + ((mine ^ in) << 4)) : "memory");
                        send(planes + ((long long)cb * col_blocks + rb) * kBlockPair);
                    }
                } else {
                    // the param: 32 x 32 values at a time, a lane to a column; this warp's half of the room
                    const double rate = lr ? (double)*lr : r.lr;
                    const float keep = (float)(1.0 - rate * r.wd * (double)t.decay), move = (float)(rate * (double)t.scale);
                    float* square = reinterpret_cast<float*>(space) + (quarter & 1) * 1024;
                    if (sender) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                    together();
#pragma unroll
                    for (int c0 = 0; c0 < 64; c0 += 32) {
                        __syncwarp();
#pragma unroll
                        for (int j = 0; j < 32; ++j) square[lane * 32 + (j ^ lane)] = v[c0 + j];
                        __syncwarp();
                        const int col = cb * kBlock + c0 + lane, row0 = rb * kBlock + (quarter & 1) * 32, rows = ok && col < t.cols ? min(32, t.rows - row0) : 0;
                        float* param = t.param + (long long)row0 * t.cols + col;
#pragma unroll
                        for (int j0 = 0; j0 < 32; j0 += 16) {
                            float old[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) old[j] = j0 + j < rows ? param[(long long)(j0 + j) * t.cols] : 0.0f;
#pragma unroll
                            for (int j = 0; j < 16; ++j)
                                if (j0 + j < rows) param[(long long)(j0 + j) * t.cols] = old[j] * keep - move * square[(j0 + j) * 32 + (lane ^ (j0 + j))];
                        }
                    }
                }
            }
            if (!last) stored = w.matrix;
        }
        say();
        if (sender) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
    if (threadIdx.x == 0 && *fail_flag) {
        atomicExch(room.failed, 1u);
        if (status) atomicExch(status, 1);
    }
}

// ---- small matrices: all of a step in one CTA ----------------------------------------------------------------
// x and A (then B in its place) stay in shared memory in the form above, sums in tensor memory, in columns of their own for every block
// of k; a product is a few instructions between two barriers.  Eight matrices of 64 to 256: 58 us, 3.9 for each of 15 products with its
// epilogue, where the launch for all matrices takes 8.  A matrix that has more rows than columns is taken as its transpose.  x: [part][block along][block across], across the shorter side.
constexpr int kSoloThreads = 512;
constexpr int kSoloBlocks = 13;                             // of x and A in both parts
constexpr int kSoloColumns = 512;                           // of tensor memory
constexpr int kSoloShared = 1024 + (2 * kSoloBlocks + 1) * kBlockBytes + 512;       // (the tensor core reads 128 rows, of 64 the next block as well)
static_assert(kSoloShared <= 227 << 10, "shared memory of a CTA");

__device__ __forceinline__ unsigned long long describe_apart(unsigned address, unsigned apart) {
    return (describe(address, 0) & ~(0x3FFFull << 16)) | (unsigned long long)(apart >> 4) << 16;
}

__global__ void __launch_bounds__(kSoloThreads, 1)
muon_solo_kernel(const void* plan, const Told told, const Rates r, const Poly poly, const float* lr, const float* grad_scale, float* step, int alone, int* status) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ double words[kSoloThreads / 32];
    __shared__ unsigned long long bar;
    __shared__ unsigned tmem_holder;
    __shared__ int fail_flag;
    const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(&bar, 1);
        fail_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) tmem_alloc(&tmem_holder, kSoloColumns);
    // Behind the launch for the other matrices, which lets this one start when all earlier kernels have ended: nothing of it is
    // waited for until the end.
    if (alone) asm volatile("griddepcontrol.wait;" ::: "memory");
    if (alone) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = (unsigned)warp_uniform((int)tmem_holder);
    if (fits(plan, told)) {
        if (alone && blockIdx.x == 0 && threadIdx.x == 0 && step) *step += 1.0f;
        const Matrix& t = matrices_of(plan)[told.matrices - told.solos + blockIdx.x];
        const bool tall = t.tall != 0;
        const int across = t.n_blocks, along = max(t.row_blocks, t.col_blocks), n = min(t.rows, t.cols), m = max(t.rows, t.cols);
        const int x_part = across * along * kBlockBytes, s_part = across * across * kBlockBytes;
        char *x = reinterpret_cast<char*>(smem), *square = x + 2 * x_part;
        const unsigned x_at = smem_u32(x), s_at = smem_u32(square);
        // The place of x(i, j) in fp32: a block's 64 x 64 values in the place of its two parts, 32 rows in either, fours of a row
        // swizzled so that neighbours by rows, and every fourth one, lie in different banks
        const auto value_at = [&](int i, int j) {
            return reinterpret_cast<float*>(x + ((j >> 6) * across + (i >> 6)) * kBlockBytes + (i & 32 ? x_part : 0)) + (i & 31) * kBlock +
                   ((((j & 63) >> 2) ^ ((i ^ (i >> 2)) & 7)) << 2) + (j & 3);
        };
        if (n < across * kBlock || m < along * kBlock) {
            for (int e = threadIdx.x; e < 2 * x_part / 16; e += kSoloThreads) reinterpret_cast<uint4*>(x)[e] = make_uint4(0, 0, 0, 0);
            __syncthreads();
        }
        // the mean, u, and the sum of its squares; values by fours where the tensors lie so
        const float s = grad_scale ? *grad_scale : 1.0f;
        const int size = t.rows * t.cols;
        const bool vec = (((uintptr_t)t.grad | (uintptr_t)t.mean | (uintptr_t)t.param) & 15) == 0;
        // all of a tensor's values, a run of them next to one another by a thread and BATCH runs at a time
        const auto walk = [&](auto&& load, auto&& use) {
            constexpr int BATCH = 4;
            const int whole = vec ? size / 4 : 0;
            for (int i0 = threadIdx.x; i0 < whole; i0 += BATCH * kSoloThreads) {
                float4 v[BATCH][2];
#pragma unroll
                for (int k = 0; k < BATCH; ++k)
                    if (i0 + k * kSoloThreads < whole) load(4 * (i0 + k * kSoloThreads), v[k], std::integral_constant<int, 4>());
#pragma unroll
                for (int k = 0; k < BATCH; ++k)
                    if (i0 + k * kSoloThreads < whole) use(4 * (i0 + k * kSoloThreads), v[k], std::integral_constant<int, 4>());
            }
            for (int i0 = 4 * whole + threadIdx.x; i0 < size; i0 += 2 * BATCH * kSoloThreads) {
                float4 v[2 * BATCH][2];
#pragma unroll
                for (int k = 0; k < 2 * BATCH; ++k)
                    if (i0 + k * kSoloThreads < size) load(i0 + k * kSoloThreads, v[k], std::integral_constant<int, 1>());
#pragma unroll
                for (int k = 0; k < 2 * BATCH; ++k)
                    if (i0 + k * kSoloThreads < size) use(i0 + k * kSoloThreads, v[k], std::integral_constant<int, 1>());
            }
        };
        const auto get = [](const float* from, float4& v, auto count) {
            if constexpr (decltype(count)::value == 4) v = *reinterpret_cast<const float4*>(from);
            else v.x = *from;
        };
        const auto put = [](float* to, const float4& v, auto count) {
            if constexpr (decltype(count)::value == 4) *reinterpret_cast<float4*>(to) = v;
            else *to = v.x;
        };
        // visits `count` values from number i on: use(j, value) may change it where it lies in fp32
        const auto places = [&](int i, auto count, auto&& use) {
            int at_row = i / t.cols, at_col = i - at_row * t.cols;
            if (decltype(count)::value == 4 && !tall && (t.cols & 3) == 0) {
                float4* four = reinterpret_cast<float4*>(value_at(at_row, at_col));
                float4 v = *four;
                use(0, v.x);
                use(1, v.y);
                use(2, v.z);
                use(3, v.w);
                *four = v;
                return;
            }
#pragma unroll
            for (int j = 0; j < decltype(count)::value; ++j) {
                use(j, *(tall ? value_at(at_col, at_row) : value_at(at_row, at_col)));
                if (++at_col == t.cols) { at_col = 0; ++at_row; }
            }
        };
        double q = 0.0;
        walk([&](int i, float4* v, auto count) {
                 get(t.grad + i, v[0], count);
                 get(t.mean + i, v[1], count);
             },
             [&](int i, float4* v, auto count) {
                 float* g = reinterpret_cast<float*>(&v[0]);
                 float* mean = reinterpret_cast<float*>(&v[1]);
                 places(i, count, [&](int j, float& value) {
                     mean[j] = r.mu * mean[j] + r.rest * (g[j] * s);
                     const float u = r.nesterov ? r.rest * (g[j] * s) + r.mu * mean[j] : mean[j];
                     value = u;
                     q = fma((double)u, (double)u, q);
                 });
                 put(t.mean + i, v[1], count);
             });
        q = cta_sum<kSoloThreads>(q, words);
        const float2 factors = over_norm(sqrt(q) + (double)r.eps, power(poly.x[0]));
        // x in parts, four blocks at a time: a thread to eight values next to one another of each
        for (int b0 = 0; b0 < across * along; b0 += 4) {
            const int in_row = threadIdx.x >> 3, piece = threadIdx.x & 7;
            float v[4][8];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                if (b0 + b >= across * along) break;
                const int i = ((b0 + b) % across) * kBlock + in_row, j = ((b0 + b) / across) * kBlock + piece * 8;
                const float4 first = *reinterpret_cast<const float4*>(value_at(i, j)), second = *reinterpret_cast<const float4*>(value_at(i, j + 4));
                const float w[8] = {first.x, first.y, first.z, first.w, second.x, second.y, second.z, second.w};
#pragma unroll
                for (int e = 0; e < 8; ++e) v[b][e] = w[e] * factors.x * factors.y;
            }
            __syncthreads();
#pragma unroll
            for (int b = 0; b < 4; ++b)
                if (b0 + b < across * along) put_piece(x + (b0 + b) * kBlockBytes, in_row, piece, v[b], x_part);
        }

        const int quarter = warp & 3, turn = warp >> 2, row = quarter * 32 + lane;     // (sixteen columns by turns of four warps)
        const bool used = row < across * kBlock;            // (of a warp all or none)
        const unsigned lanes = tmem + ((unsigned)(quarter * 32) << 16);
        unsigned parity = 0;
        // what has been stored is there for the tensor core; `issue` by one thread; its results are there for everybody
        const auto products = [&](auto&& issue) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            tc_fence_before();
            __syncthreads();
            if (warp == 0 && elect_one()) {
                tc_fence_after();
                issue();
                tc_commit(&bar);
            }
            __syncwarp();
            if (!mbar_wait(&bar, parity)) atomicExch(&fail_flag, 1);
            parity ^= 1u;
            tc_fence_after();
        };
        // three products of parts, the small ones first, of 64 of k
        const auto three = [&](unsigned sum, unsigned p, unsigned p_part, unsigned long long q_hi, unsigned q_part, unsigned q_step, unsigned instruction, bool more) {
            const unsigned long long p_hi = describe(p, 0), p_lo = describe(p + p_part, 0), q_lo = q_hi + (q_part >> 4);
            for (int k = 0; k < 4; ++k) multiply_f16(sum, p_hi + 2 * k, q_lo + k * q_step, instruction, more || k > 0);
            for (int k = 0; k < 4; ++k) multiply_f16(sum, p_lo + 2 * k, q_hi + k * q_step, instruction, 1);
            for (int k = 0; k < 4; ++k) multiply_f16(sum, p_hi + 2 * k, q_hi + k * q_step, instruction, 1);
        };
        const auto instruction_of = [](int width, unsigned q_major) { return (1u << 4) | (q_major << 16) | ((unsigned)(width >> 3) << 17) | ((128u >> 4) << 24); };
        // sixteen columns of `count` sums that lie `apart`, two sums at a time
        const auto columns = [&](unsigned from, int count, int apart, float* v) {
            unsigned w[2][16];
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = 0.0f;
            for (int b = 0; b < count; b += 2) {
                tmem_ld16(lanes + from + b * apart, w[0]);
                if (b + 1 < count) tmem_ld16(lanes + from + (b + 1) * apart, w[1]);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] += __uint_as_float(w[0][j]);
                if (b + 1 < count)
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] += __uint_as_float(w[1][j]);
            }
        };
        const auto put_columns = [&](char* first, int col, const float* v, int part) {
            char* block = first + ((col >> 6) * across + (row >> 6)) * kBlockBytes;
            put_piece(block, row & 63, (col & 63) >> 3, v, part);
            put_piece(block, row & 63, ((col & 63) >> 3) + 1, v + 8, part);
        };
        const int side = across * kBlock, per_sum = (along * side + kSoloColumns - 1) / kSoloColumns, sums = (along + per_sum - 1) / per_sum;
        const int chunk = kSoloColumns / across;            // columns of x that are multiplied at a time
        const double rate = lr ? (double)*lr : r.lr;
        const float keep = (float)(1.0 - rate * r.wd * (double)t.decay), move = (float)(rate * (double)t.scale);
        for (int k = 0; k < poly.steps; ++k) {
            const bool last = k == poly.steps - 1;
            float held[32];                                 // this thread's part of A
            products([&] {
                for (int b = 0; b < along; ++b) {
                    const unsigned at = x_at + b * across * kBlockBytes;
                    three(tmem + b / per_sum * side, at, x_part, describe(at, 0), x_part, 2, instruction_of(side, 0), b % per_sum > 0);
                }
            });
            if (used) {
                const float factor = power(poly.square[k] - 2 * poly.x[k]);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    if (c >= across) continue;
                    const int col = (4 * c + turn) * 16;
                    float* v = held + 16 * c;
                    columns(col, sums, side, v);
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] *= factor;
                    put_columns(square, col, v, s_part);
                }
            }
            products([&] {
                for (int b = 0; b < across; ++b) {
                    const unsigned at = s_at + b * across * kBlockBytes;
                    three(tmem + b * side, at, s_part, describe(at, 0), s_part, 2, instruction_of(side, 0), false);
                }
            });
            if (used) {
                const float factor = poly.c * power(poly.poly[k] - 2 * poly.square[k]), linear = poly.b * power(poly.poly[k] - poly.square[k]);
                const float diagonal = poly.a * power(poly.poly[k]);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    if (c >= across) continue;
                    const int col = (4 * c + turn) * 16;
                    float v[16];
                    columns(col, across, side, v);
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        v[j] = fmaf(linear, held[16 * c + j], factor * v[j]);
                        if (row == col + j && row < n) v[j] += diagonal;
                    }
                    put_columns(square, col, v, s_part);
                }
            }
            for (int c0 = 0; c0 < along * kBlock; c0 += chunk) {
                const int width = min(chunk, along * kBlock - c0);
                products([&] {
                    for (int b = 0; b < across; ++b)
                        for (int w0 = 0; w0 < width; w0 += 256) {
                            const unsigned at = x_at + (((c0 + w0) >> 6) * across + b) * kBlockBytes;
                            three(tmem + b * chunk + w0, s_at + b * across * kBlockBytes, s_part, describe_apart(at, across * kBlockBytes), x_part, 2048 >> 4,
                                  instruction_of(min(256, width - w0), 1), false);
                        }
                });
                // (the products have been made: their operand's place is free)
                if (used) {
                    const float factor = last ? power(-poly.x[k] - poly.poly[k]) : power(poly.x[k + 1] - poly.x[k] - poly.poly[k]);
#pragma unroll 2
                    for (int w0 = turn * 16; w0 < width; w0 += 64) {
                        float v[16];
                        columns(w0, across, chunk, v);
#pragma unroll
                        for (int j = 0; j < 16; ++j) v[j] *= factor;
                        const int col = c0 + w0;
                        if (!last) {
                            put_columns(x, col, v, x_part);
                        } else if (row < n) {
#pragma unroll
                            for (int j = 0; j < 16; j += 4) *reinterpret_cast<float4*>(value_at(row, col + j)) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                        }
                    }
                }
            }
            if (last) {
                __syncthreads();
                walk([&](int i, float4* v, auto count) { get(t.param + i, v[0], count); },
                     [&](int i, float4* v, auto count) {
                         float* p = reinterpret_cast<float*>(&v[0]);
                         places(i, count, [&](int j, const float& value) { p[j] = p[j] * keep - move * value; });
                         put(t.param + i, v[0], count);
                     });
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, kSoloColumns);
    }
    if (threadIdx.x == 0 && fail_flag && status) atomicExch(status, 1);
    if (!alone) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    }
}

int check_matrices(const b2_muon_matrix* list, int count) {
    B2_REQUIRE(count >= 0 && (count == 0 || list), "bad list of matrices");
    for (int i = 0; i < count; ++i) {
        const b2_muon_matrix& t = list[i];
        B2_REQUIRE(t.rows >= 0 && t.cols >= 0 && t.rows <= kMostSide && t.cols <= kMostSide && (t.rows < t.cols ? t.rows : t.cols) <= kMostShort,
                   "matrix %d is %lld x %lld: sides of at most %lld, the shorter one of %lld", i, (long long)t.rows, (long long)t.cols, kMostSide, kMostShort);
        if (t.rows == 0 || t.cols == 0) continue;
        B2_REQUIRE(t.param && t.grad && t.mean, "matrix %d: missing address", i);
        B2_REQUIRE((((uintptr_t)t.param | (uintptr_t)t.grad | (uintptr_t)t.mean) & 3) == 0, "matrix %d lies between two addresses", i);
        B2_REQUIRE(std::isfinite(t.decay) && std::isfinite(t.scale), "matrix %d: decay %g, scale %g", i, t.decay, t.scale);
    }
    return B2_OK;
}

constexpr int blocks_in(long long n) { return (int)((n + kBlock - 1) / kBlock); }

// The tiles of a product of rb x cb blocks, upper triangle alone where `half`: [i, j, width]
template <typename F>
void tiles_of(int rb, int cb, bool half, int width, F&& tile) {
    for (int i = 0; 2 * i < rb; ++i)
        for (int j = half ? 2 * i : 0; j < cb; j += width) tile(i, j, std::min(width, cb - j));
}

// Cycles of an item, as measured: blocks of k, which wait for shared memory (64 columns want 72 KB read and 48 KB written a block at 128
// bytes a cycle, 256 columns 144 and 96), and what starts and ends it (lists of 8 to 48 matrices of 64 to 8192 took as long with 4000,
// 12000 and 20000 for that).
double cycles_of(int width, int k_blocks) {
    static const double block[5] = {0, 1150, 1430, 1700, 1960};
    return block[width] * k_blocks + 8000;
}

Layout layout_of(const b2_muon_matrix* list, int count) {
    Layout found;
    long long at = 0;
    const auto take = [&](long long blocks) {
        const long long from = at;
        at += blocks * kBlockPair;
        return from;
    };
    for (int i = 0; i < count; ++i) {
        const b2_muon_matrix& s = list[i];
        if (s.rows == 0 || s.cols == 0) continue;
        Matrix t = {};
        t.param = s.param;
        t.grad = s.grad;
        t.mean = s.mean;
        t.rows = (int)s.rows;
        t.cols = (int)s.cols;
        t.tall = t.rows > t.cols;
        t.decay = s.decay;
        t.scale = s.scale;
        t.row_blocks = blocks_in(t.rows);
        t.col_blocks = blocks_in(t.cols);
        t.n_blocks = std::min(t.row_blocks, t.col_blocks);
        found.matrices.push_back(t);
    }
    // long sums first: the last items of a phase are short ones
    std::stable_sort(found.matrices.begin(), found.matrices.end(),
                     [](const Matrix& a, const Matrix& b) { return std::max(a.row_blocks, a.col_blocks) > std::max(b.row_blocks, b.col_blocks); });
    const auto rest = std::stable_partition(found.matrices.begin(), found.matrices.end(), [](const Matrix& t) {
        return (long long)t.row_blocks * t.col_blocks + (long long)t.n_blocks * t.n_blocks > kSoloBlocks;
    });
    found.solos = found.matrices.end() - rest;
    const size_t shared = rest - found.matrices.begin();     // matrices that share the launch for all
    for (int index = 0; index < (int)shared; ++index) {
        Matrix& t = found.matrices[index];
        const long long size = (long long)t.rows * t.cols, blocks = (long long)t.row_blocks * t.col_blocks;
        t.x[0] = take(blocks);
        t.x[1] = take(blocks);
        t.square = take((long long)t.n_blocks * t.n_blocks);
        t.poly = take((long long)t.n_blocks * t.n_blocks);
        t.held = take((long long)t.n_blocks * t.n_blocks);
        t.first_chunk = (int)found.chunks.size();
        const long long each = std::max(2048ll, (size / 512 + 2047) / 2048 * 2048);
        for (long long k = 0; k < size; k += each) found.chunks.push_back({index, (int)std::min(each, size - k), k});
        t.chunks = (int)found.chunks.size() - t.first_chunk;
        for (int k = 0; k < blocks; ++k) found.blocks.push_back({index, k});
    }
    // Groups of matrices whose phases keep the machine busy while another's end: some three tiles to an SM or more, in groups of one
    // size (a last group of few matrices would wait for each of its phases).  48 matrices of 640 to 2560 and 8 of 2048 to 8192: 3.23 and 12.5
    // ms with half a tile to an SM, 2.95 and 11.4 with one, 2.93 and 11.1 with two, 2.94 and 11.1 with three
    const auto tiles_in = [&](size_t m) {
        long long tiles = 0;
        tiles_of(found.matrices[m].n_blocks, found.matrices[m].n_blocks, true, 4, [&](int, int, int) { ++tiles; });
        return tiles;
    };
    long long tiles_left = 0;
    for (size_t m = 0; m < shared; ++m) tiles_left += tiles_in(m);
    long long groups_left = std::max(1ll, tiles_left / (3 * b2::kSms));
    for (size_t from = 0; from < shared; --groups_left) {
        size_t to = from;
        const long long enough = tiles_left / std::max(1ll, groups_left);
        for (long long tiles = 0; to < shared && (to == from || tiles < enough || groups_left <= 1); ++to) {
            tiles += tiles_in(to);
            tiles_left -= tiles_in(to);
        }
        const long long first = (long long)found.items.size();
        for (int phase = GRAM; phase <= MULTIPLY; ++phase) {
            // the width of tiles that ends the phase first, by its longest item and by all of them
            int best = 4;
            double least = 1e300;
            for (int width : {4, 2, 1}) {
                double all = 0, longest = 0;
                for (size_t m = from; m < to; ++m) {
                    const Matrix& t = found.matrices[m];
                    const int k_blocks = phase == GRAM ? std::max(t.row_blocks, t.col_blocks) : t.n_blocks;
                    tiles_of(phase == MULTIPLY ? t.row_blocks : t.n_blocks, phase == MULTIPLY ? t.col_blocks : t.n_blocks, phase != MULTIPLY, width, [&](int, int, int w) {
                        all += cycles_of(w, k_blocks);
                        longest = std::max(longest, cycles_of(w, k_blocks));
                    });
                }
                const double end = std::max(all / b2::kSms, longest);
                if (end < least * 0.97) {
                    least = end;
                    best = width;
                }
            }
            for (size_t m = from; m < to; ++m) {
                Matrix& t = found.matrices[m];
                const size_t before = found.items.size();
                tiles_of(phase == MULTIPLY ? t.row_blocks : t.n_blocks, phase == MULTIPLY ? t.col_blocks : t.n_blocks, phase != MULTIPLY, best,
                         [&](int i, int j, int w) { found.items.push_back({(int)m, (short)phase, (short)w, i, j}); });
                t.items[phase] = (int)(found.items.size() - before);
            }
        }
        found.groups.push_back({first, (long long)found.items.size() - first});
        from = to;
    }
    found.bytes = at;
    return found;
}

size_t counter_bytes(const b2_muon_sizes& s) { return ((size_t)s.chunks * 8 + 16 + (size_t)s.matrices * 4 + 1023) / 1024 * 1024; }

int sizes_of(const Layout& l, b2_muon_sizes* s) {
    s->plan_bytes = l.plan_bytes() + 64;
    s->matrices = (int64_t)l.matrices.size();
    s->chunks = (int64_t)l.chunks.size();
    s->items = (int64_t)l.items.size();
    s->blocks = (int64_t)l.blocks.size();
    s->solos = (int64_t)l.solos;
    s->scratch_bytes = counter_bytes(*s) + (size_t)l.bytes + 1024;
    return B2_OK;
}

// The largest values that |p| and |p(s) / s| have over [0, top]: at the ends, where p' = a + 3 b t + 5 c t^2 is zero, t = s^2, and where
// a + b t + c t^2 turns
void reach(double a, double b, double c, double top, double* of_p, double* of_factor) {
    double at[5] = {0.0, top * top, 0.0, 0.0, 0.0};
    if (c != 0.0) {
        const double inside = 9.0 * b * b - 20.0 * a * c, root = inside > 0.0 ? std::sqrt(inside) : 0.0;
        at[2] = (-3.0 * b + root) / (10.0 * c);
        at[3] = (-3.0 * b - root) / (10.0 * c);
        at[4] = -b / (2.0 * c);
    } else if (b != 0.0) {
        at[2] = -a / (3.0 * b);
    }
    *of_p = *of_factor = 0.0;
    for (double t : at) {
        if (!(t >= 0.0 && t <= top * top)) continue;
        const double f = std::fabs(a + (b + c * t) * t);
        *of_factor = std::max(*of_factor, f);
        *of_p = std::max(*of_p, std::sqrt(t) * f);
    }
}
// The power of two that takes values up to `most` next to fp16's largest, 65504; a value that is no larger than its operand's largest
// singular value, 1 % of rounding included, stays below 60000
int exponent_of(double most) {
    int e;
    std::frexp(60000.0 / (1.01 * most + 1e-30), &e);
    return std::max(-30, std::min(20, e - 1));
}

char* aligned(void* p, size_t to) { return (char*)(((uintptr_t)p + to - 1) / to * to); }

// Blocks write in any order: what one writes no other may read or write.
int check_alone(const b2_muon_matrix* list, int count, const void* plan, size_t plan_bytes) {
    struct Range {
        uintptr_t from, to;
        bool operator<(const Range& o) const { return from < o.from; }
    };
    const auto range = [](const void* p, size_t bytes) { return Range{(uintptr_t)p, (uintptr_t)p + bytes}; };
    std::vector<Range> written = {range(plan, plan_bytes)};
    for (int i = 0; i < count; ++i) {
        const size_t bytes = (size_t)list[i].rows * list[i].cols * 4;
        if (!bytes) continue;
        written.push_back(range(list[i].param, bytes));
        written.push_back(range(list[i].mean, bytes));
    }
    std::sort(written.begin(), written.end());
    for (size_t k = 1; k < written.size(); ++k)
        B2_REQUIRE(written[k - 1].to <= written[k].from, "matrices of the plan overlap, or lie in its memory");
    for (int i = 0; i < count; ++i) {
        const size_t bytes = (size_t)list[i].rows * list[i].cols * 4;
        if (!bytes) continue;
        const Range g = range(list[i].grad, bytes);
        const auto next = std::lower_bound(written.begin(), written.end(), Range{g.to, 0});     // the first that begins behind it
        B2_REQUIRE(next == written.begin() || (next - 1)->to <= g.from, "gradient %d overlaps a matrix that the step writes", i);
    }
    return B2_OK;
}

}  // namespace

extern "C" int b2_muon_plan_sizes(const b2_muon_matrix* list, int32_t count, b2_muon_sizes* sizes) {
    B2_REQUIRE(sizes, "missing argument");
    B2_CHECK(check_matrices(list, count));
    try {
        return sizes_of(layout_of(list, count), sizes);
    } catch (const std::bad_alloc&) {
        return b2::fail(B2_ERR_INVALID, "no memory for a plan of %d matrices", count);
    }
}

extern "C" int b2_muon_plan_tiles(const b2_muon_matrix* list, int32_t count, b2_muon_tiles* tiles) {
    B2_REQUIRE(tiles, "missing argument");
    B2_CHECK(check_matrices(list, count));
    try {
        const Layout l = layout_of(list, count);
        *tiles = {};
        tiles->groups = (int64_t)l.groups.size();
        for (const Item& item : l.items) ++tiles->tiles[item.phase][item.width - 1];
    } catch (const std::bad_alloc&) {
        return b2::fail(B2_ERR_INVALID, "no memory for a plan of %d matrices", count);
    }
    return B2_OK;
}

extern "C" int b2_muon_launches(const b2_muon_sizes* s, int32_t* launches) {
    B2_REQUIRE(s && launches, "missing argument");
    *launches = (s->items > 0 ? 3 : 0) + (s->solos > 0 ? 1 : 0);
    if (*launches == 0) *launches = 1;               // (the number of the step)
    return B2_OK;
}

extern "C" int b2_muon_plan(const b2_muon_matrix* list, int32_t count, void* plan, size_t plan_bytes, void* stream) {
    B2_CHECK(check_matrices(list, count));
    try {
        const Layout l = layout_of(list, count);
        b2_muon_sizes s;
        B2_CHECK(sizes_of(l, &s));
        B2_REQUIRE(plan && plan_bytes >= s.plan_bytes, "the plan needs %zu bytes, got %zu", s.plan_bytes, plan_bytes);
        B2_CHECK(check_alone(list, count, plan, s.plan_bytes));
        b2::Memory memory;
        B2_CHECK(memory.find_device());
        B2_CHECK(memory.written(plan, "the plan"));
        for (int i = 0; i < count; ++i) {
            if (list[i].rows == 0 || list[i].cols == 0) continue;
            B2_CHECK(memory.written(list[i].param, "a matrix of the plan"));
            B2_CHECK(memory.read(list[i].grad, "a gradient of the plan"));
            B2_CHECK(memory.written(list[i].mean, "a mean of the plan"));
        }
        cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
        B2_CUDA(cudaStreamIsCapturing((cudaStream_t)stream, &capturing));
        B2_REQUIRE(capturing == cudaStreamCaptureStatusNone, "a plan is made before its stream is captured");
        std::vector<char> host(l.plan_bytes(), 0);
        *reinterpret_cast<Header*>(host.data()) = {s.matrices, s.chunks, s.items, s.blocks, s.solos, (long long)s.scratch_bytes, (long long)l.groups.size()};
        char* to = host.data() + kHeader;
        const auto put = [&](const void* from, size_t bytes) {
            std::copy((const char*)from, (const char*)from + bytes, to);
            to += bytes;
        };
        put(l.matrices.data(), l.matrices.size() * sizeof(Matrix));
        put(l.chunks.data(), l.chunks.size() * sizeof(Chunk));
        put(l.blocks.data(), l.blocks.size() * sizeof(Block));
        put(l.items.data(), l.items.size() * sizeof(Item));
        put(l.groups.data(), l.groups.size() * sizeof(Group));
        // (pageable memory: the copy has been staged when the call returns)
        B2_CUDA(cudaMemcpyAsync(aligned(plan, 64), host.data(), host.size(), cudaMemcpyHostToDevice, (cudaStream_t)stream));
        B2_CUDA(cudaStreamSynchronize((cudaStream_t)stream));
    } catch (const std::bad_alloc&) {
        return b2::fail(B2_ERR_INVALID, "no memory for a plan of %d matrices", count);
    }
    return B2_OK;
}

extern "C" int b2_muon_step(void* plan, const b2_muon_sizes* s, const b2_muon_hyper* h, const float* lr, const float* grad_scale, float* step, void* scratch,
                            size_t scratch_bytes, int32_t* status, void* stream) {
    B2_REQUIRE(plan && s && h && s->matrices >= 0 && s->chunks >= 0 && s->items >= 0 && s->blocks >= 0 && s->solos >= 0 && s->solos <= s->matrices, "bad argument");
    B2_REQUIRE(scratch && scratch_bytes >= s->scratch_bytes, "the step needs %zu bytes of scratch, got %zu", s->scratch_bytes, scratch_bytes);
    B2_REQUIRE(std::isfinite(h->lr) && h->momentum >= 0.0 && h->momentum < 1.0 && std::isfinite(h->eps) && h->eps >= 0.0 && std::isfinite(h->weight_decay),
               "bad rates: lr %g, momentum %g, eps %g, weight decay %g", h->lr, h->momentum, h->eps, h->weight_decay);
    B2_REQUIRE(h->steps >= 1 && h->steps <= kMostSteps && std::isfinite(h->a) && std::isfinite(h->b) && std::isfinite(h->c), "bad polynomial: %d steps of %g, %g, %g",
               h->steps, h->a, h->b, h->c);
    B2_REQUIRE((((uintptr_t)lr | (uintptr_t)grad_scale | (uintptr_t)step | (uintptr_t)status) & 3) == 0, "a number of the step lies between two addresses");
    B2_REQUIRE(!b2::overlap(plan, s->plan_bytes, scratch, s->scratch_bytes), "the plan lies in the scratch");
    for (const void* number : {(const void*)lr, (const void*)grad_scale, (const void*)step, (const void*)status})
        B2_REQUIRE(!b2::overlap(number, 4, plan, s->plan_bytes) && !b2::overlap(number, 4, scratch, s->scratch_bytes),
                   "a number of the step lies in the plan or the scratch");
    for (const void* number : {(const void*)lr, (const void*)grad_scale, (const void*)status})
        B2_REQUIRE(!b2::overlap(step, 4, number, 4), "the number of the step lies in the place of another");
    B2_REQUIRE(!b2::overlap(status, 4, lr, 4) && !b2::overlap(status, 4, grad_scale, 4), "the status lies in the place of a number of the step");
    b2::Memory memory;
    B2_CHECK(memory.find_device());
    B2_CHECK(memory.written(plan, "the plan"));
    B2_CHECK(memory.written(scratch, "the scratch"));
    if (step) B2_CHECK(memory.written(step, "the number of the step"));
    if (status) B2_CHECK(memory.written(status, "the status"));
    B2_CHECK(memory.read(lr, "the rate"));
    B2_CHECK(memory.read(grad_scale, "the scale of the gradients"));
    Rates r;
    r.mu = (float)h->momentum;
    r.rest = (float)(1.0 - h->momentum);
    r.eps = (float)h->eps;
    r.lr = h->lr;
    r.wd = h->weight_decay;
    r.nesterov = h->nesterov != 0;
    Poly p = {(float)h->a, (float)h->b, (float)h->c, h->steps, {}, {}, {}};
    double top = 1.0;
    for (int k = 0; k < h->steps; ++k) {
        double next, factor;
        reach(h->a, h->b, h->c, top, &next, &factor);
        B2_REQUIRE(next <= 1e6 && factor <= 1e6, "the polynomial of %g, %g, %g takes singular values to %g in step %d", h->a, h->b, h->c, std::max(next, factor), k + 1);
        p.x[k] = (signed char)exponent_of(top);
        p.square[k] = (signed char)exponent_of(top * top);
        p.poly[k] = (signed char)exponent_of(factor);
        top = 1.001 * next;
    }
    p.x[h->steps] = (signed char)exponent_of(top);
    B2_REQUIRE(s->items <= (1ll << 30) / h->steps, "%lld items of %d steps", (long long)s->items, h->steps);
    cudaStream_t st = (cudaStream_t)stream;
    const void* base = aligned(plan, 64);
    Room room;
    char* at = aligned(scratch, 1024);
    room.sums = (double*)at;
    room.next = (unsigned*)(at + (size_t)s->chunks * 8);
    room.failed = room.next + 1;
    room.done = room.next + 4;
    room.planes = at + counter_bytes(*s);
    const Told told = {s->matrices, s->chunks, s->items, s->blocks, s->solos, (long long)s->scratch_bytes};
    const auto grid = [](long long work, long long most) { return dim3((unsigned)(work < 1 ? 1 : work < most ? work : most)); };
    static std::atomic<unsigned long long> done{0}, done_solo{0};
    if (s->items > 0 || s->solos == 0)
        B2_CUDA((b2::launch_after(muon_mean_kernel, grid(s->chunks, b2::kSms * 8), kMeanThreads, 0, st, base, told, r, grad_scale, step, room)));
    if (s->items > 0) {
        B2_CUDA((b2::launch_after(muon_parts_kernel, grid(s->blocks, b2::kSms * 8), kMeanThreads, 0, st, base, told, r, grad_scale, (int)p.x[0], room)));
        B2_CHECK(b2::allow_shared((const void*)muon_product_kernel, kProductShared, &done));
        // (SMs for the small matrices where few items would leave some idle anyway: these need 58 us, which would come on top)
        const long long left = s->items < 8 * b2::kSms ? b2::kSms - std::min<long long>(s->solos, 8) : b2::kSms;
        B2_CUDA((b2::launch_after(muon_product_kernel, grid(s->items, left), kProductThreads, (size_t)kProductShared, st, base, told, r, p, lr, room, status)));
    }
    if (s->solos > 0) {
        B2_CHECK(b2::allow_shared((const void*)muon_solo_kernel, kSoloShared, &done_solo));
        B2_CUDA((b2::launch_after(muon_solo_kernel, grid(s->solos, 1 << 30), kSoloThreads, (size_t)kSoloShared, st, base, told, r, p, lr, grad_scale, step,
                                  (int)(s->items == 0), status)));
    }
    return B2_OK;
}
