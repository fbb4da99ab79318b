// One optimizer step over many matrices whose updates are orthogonalised:
//
//   mean = mu mean + (1 - mu) g,  u = (1 - mu) g + mu mean,  x = u / (|u| + eps)
//   `steps` times:  A = x x^T,  B = b A + c A A,  x = a x + B x
//   param = param (1 - lr wd decay) - lr scale x
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <new>
#include <vector>

#include "b2_operators.h"

namespace {

constexpr int kThreads = 256;
constexpr int kTile = 64, kDepth = 16;
constexpr int kMostSteps = 100;
constexpr long long kMostSide = 1 << 20, kMostShort = 1 << 15;

// One matrix.  Offsets are values of the scratch, from its aligned start on.
struct Matrix {
    float* param;
    const float* grad;
    float* mean;
    long long x[2], square, poly;            // two turns of x [rows][cols], A and B [n][n]
    int rows, cols, n, m;                    // n, m: the shorter and the longer side
    int first_chunk, chunks;
    float decay, scale;
};
struct Chunk {
    int matrix, n;
    long long at;
};
struct Item {
    int matrix;
    int i, j;
};
struct Header {
    long long matrices, chunks, items;
    long long squares, products;             // items of a product n x n, and of one with x
};
constexpr size_t kHeader = 64;

struct Layout {
    std::vector<Matrix> matrices;
    std::vector<Chunk> chunks;
    std::vector<Item> squares, products;
    long long values;                        // of the scratch
    size_t plan_bytes() const {
        return kHeader + matrices.size() * sizeof(Matrix) + chunks.size() * sizeof(Chunk) + (squares.size() + products.size()) * sizeof(Item);
    }
};

struct Rates {
    float mu, rest, eps, a, b, c;
    double lr, wd;
    int nesterov;
};

__device__ __forceinline__ const Header* header_of(const void* plan) { return static_cast<const Header*>(plan); }
__device__ __forceinline__ const Matrix* matrices_of(const void* plan) { return reinterpret_cast<const Matrix*>(static_cast<const char*>(plan) + kHeader); }
__device__ __forceinline__ const Chunk* chunks_of(const void* plan) { return reinterpret_cast<const Chunk*>(matrices_of(plan) + header_of(plan)->matrices); }
__device__ __forceinline__ const Item* items_of(const void* plan) { return reinterpret_cast<const Item*>(chunks_of(plan) + header_of(plan)->chunks); }
__device__ __forceinline__ bool fits(const void* plan, long long matrices, long long chunks, long long items) {
    const Header* h = header_of(plan);
    return h->matrices == matrices && h->chunks == chunks && h->items == items;
}

// u of a chunk, to the first turn of x, the mean, and the sum of squares in 64 bits
__global__ void __launch_bounds__(kThreads)
muon_mean_kernel(const void* plan, long long matrices, long long chunks, long long items, const Rates r, const float* grad_scale, float* step,
                 double* sums, float* scratch) {
    __shared__ double words[kThreads / 32];
    after_earlier_kernels();
    if (!fits(plan, matrices, chunks, items)) return;
    if (blockIdx.x == 0 && threadIdx.x == 0 && step) *step += 1.0f;
    const float s = grad_scale ? *grad_scale : 1.0f;
    for (long long k = blockIdx.x; k < chunks; k += gridDim.x) {
        const Chunk c = chunks_of(plan)[k];
        const Matrix& t = matrices_of(plan)[c.matrix];
        double q = 0.0;
        for (int i = threadIdx.x; i < c.n; i += kThreads) {
            const float g = t.grad[c.at + i] * s, m = r.mu * t.mean[c.at + i] + r.rest * g;
            const float u = r.nesterov ? r.rest * g + r.mu * m : m;
            t.mean[c.at + i] = m;
            scratch[t.x[0] + c.at + i] = u;
            q = fma((double)u, (double)u, q);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) words[threadIdx.x >> 5] = q;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < kThreads / 32; ++w) q += words[w];
            sums[k] = q;
        }
    }
}

__global__ void __launch_bounds__(kThreads)
muon_scale_kernel(const void* plan, long long matrices, long long chunks, long long items, float eps, const double* sums, float* scratch) {
    __shared__ double words[kThreads / 32];
    after_earlier_kernels();
    if (!fits(plan, matrices, chunks, items)) return;
    for (long long k = blockIdx.x; k < chunks; k += gridDim.x) {
        const Chunk c = chunks_of(plan)[k];
        const Matrix& t = matrices_of(plan)[c.matrix];
        double q = 0.0;
        for (int i = threadIdx.x; i < t.chunks; i += kThreads) q += sums[t.first_chunk + i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) words[threadIdx.x >> 5] = q;
        __syncthreads();
        q = 0.0;
        for (int w = 0; w < kThreads / 32; ++w) q += words[w];
        const float inverse = (float)(1.0 / (sqrt(q) + (double)eps));
        for (int i = threadIdx.x; i < c.n; i += kThreads) scratch[t.x[0] + c.at + i] *= inverse;
    }
}

// A tile of one product.  phase 0: A = x x^T (x^T x), 1: B = b A + c A A, 2: x = a x + B x (x B), the last of which moves the
// param instead.  P [rows of the tile][k], Q [k][columns], by strides.
__global__ void __launch_bounds__(kThreads)
muon_product_kernel(const void* plan, long long matrices, long long chunks, long long items, int phase, int turn, int last, const Rates r, const float* lr,
                    float* scratch) {
    __shared__ float p_tile[kDepth][kTile + 4], q_tile[kDepth][kTile + 4];
    after_earlier_kernels();
    if (!fits(plan, matrices, chunks, items)) return;
    if (blockIdx.x >= (phase == 2 ? header_of(plan)->products : header_of(plan)->squares)) return;
    const Item item = items_of(plan)[(phase == 2 ? header_of(plan)->squares : 0) + blockIdx.x];
    const Matrix& t = matrices_of(plan)[item.matrix];
    const bool tall = t.rows > t.cols;
    const float *x = scratch + t.x[turn], *square = scratch + t.square, *poly = scratch + t.poly;
    const float *P, *Q;
    long long p_row, p_k, q_k, q_col;
    int M = t.n, N = t.n, K = t.n;
    if (phase == 0) {
        P = Q = x;
        K = t.m;
        p_row = q_col = tall ? 1 : t.cols;
        p_k = q_k = tall ? t.cols : 1;
    } else if (phase == 1) {
        P = Q = square;
        p_row = q_k = t.n;
        p_k = q_col = 1;
    } else {
        M = t.rows;
        N = t.cols;
        P = tall ? x : poly;
        Q = tall ? poly : x;
        p_row = tall ? t.cols : t.n;
        q_k = tall ? t.n : t.cols;
        p_k = q_col = 1;
    }
    const int m0 = item.i * kTile, n0 = item.j * kTile;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float sum[4][4] = {};
    for (int k0 = 0; k0 < K; k0 += kDepth) {
        for (int e = threadIdx.x; e < kTile * kDepth; e += kThreads) {
            // neighbours in memory to neighbouring threads
            const int a = p_k == 1 ? e / kDepth : e % kTile, ka = p_k == 1 ? e % kDepth : e / kTile;
            p_tile[ka][a] = m0 + a < M && k0 + ka < K ? P[(m0 + a) * p_row + (k0 + ka) * p_k] : 0.0f;
            const int b = q_k == 1 ? e / kDepth : e % kTile, kb = q_k == 1 ? e % kDepth : e / kTile;
            q_tile[kb][b] = n0 + b < N && k0 + kb < K ? Q[(k0 + kb) * q_k + (n0 + b) * q_col] : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kDepth; ++k) {
            float u[4], v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                u[j] = p_tile[k][ty * 4 + j];
                v[j] = q_tile[k][tx * 4 + j];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[i][j] = fmaf(u[i], v[j], sum[i][j]);
        }
        __syncthreads();
    }
    const double rate = lr ? (double)*lr : r.lr;
    const float keep = (float)(1.0 - rate * r.wd * (double)t.decay), move = (float)(rate * (double)t.scale);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const long long row = m0 + ty * 4 + i, col = n0 + tx * 4 + j;
            if (row >= M || col >= N) continue;
            const long long at = row * N + col;
            if (phase == 0) scratch[t.square + at] = sum[i][j];
            else if (phase == 1) scratch[t.poly + at] = fmaf(r.b, square[at], r.c * sum[i][j]);
            else {
                const float y = fmaf(r.a, x[at], sum[i][j]);
                if (!last) scratch[t.x[turn ^ 1] + at] = y;
                else t.param[at] = t.param[at] * keep - move * y;
            }
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

Layout layout_of(const b2_muon_matrix* list, int count) {
    Layout found;
    long long at = 0;
    const auto take = [&](long long n) {
        const long long from = at;
        at += (n + 63) / 64 * 64;
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
        t.n = std::min(t.rows, t.cols);
        t.m = std::max(t.rows, t.cols);
        t.decay = s.decay;
        t.scale = s.scale;
        const long long size = s.rows * s.cols;
        t.x[0] = take(size);
        t.x[1] = take(size);
        t.square = take((long long)t.n * t.n);
        t.poly = take((long long)t.n * t.n);
        t.first_chunk = (int)found.chunks.size();
        const long long each = std::max(2048ll, (size / 512 + 2047) / 2048 * 2048);
        const int index = (int)found.matrices.size();
        for (long long k = 0; k < size; k += each) found.chunks.push_back({index, (int)std::min(each, size - k), k});
        t.chunks = (int)found.chunks.size() - t.first_chunk;
        for (int a = 0; a < (t.n + kTile - 1) / kTile; ++a)
            for (int b = 0; b < (t.n + kTile - 1) / kTile; ++b) found.squares.push_back({index, a, b});
        for (int a = 0; a < (t.rows + kTile - 1) / kTile; ++a)
            for (int b = 0; b < (t.cols + kTile - 1) / kTile; ++b) found.products.push_back({index, a, b});
        found.matrices.push_back(t);
    }
    found.values = at;
    return found;
}

// The scratch: sums of squares, and behind them the values
size_t sums_bytes(long long chunks) { return ((size_t)chunks * 8 + 255) / 256 * 256; }

int sizes_of(const Layout& l, b2_muon_sizes* s) {
    s->plan_bytes = l.plan_bytes() + 64;
    s->scratch_bytes = sums_bytes((long long)l.chunks.size()) + (size_t)l.values * 4 + 256;
    s->matrices = (int64_t)l.matrices.size();
    s->chunks = (int64_t)l.chunks.size();
    s->items = (int64_t)(l.squares.size() + l.products.size());
    return B2_OK;
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
        *reinterpret_cast<Header*>(host.data()) = {s.matrices, s.chunks, s.items, (long long)l.squares.size(), (long long)l.products.size()};
        char* to = host.data() + kHeader;
        const auto put = [&](const void* from, size_t bytes) {
            std::copy((const char*)from, (const char*)from + bytes, to);
            to += bytes;
        };
        put(l.matrices.data(), l.matrices.size() * sizeof(Matrix));
        put(l.chunks.data(), l.chunks.size() * sizeof(Chunk));
        put(l.squares.data(), l.squares.size() * sizeof(Item));
        put(l.products.data(), l.products.size() * sizeof(Item));
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
    B2_REQUIRE(plan && s && h && s->matrices >= 0 && s->chunks >= 0 && s->items >= 0, "bad argument");
    B2_REQUIRE(scratch && scratch_bytes >= s->scratch_bytes, "the step needs %zu bytes of scratch, got %zu", s->scratch_bytes, scratch_bytes);
    B2_REQUIRE(std::isfinite(h->lr) && h->momentum >= 0.0 && h->momentum < 1.0 && std::isfinite(h->eps) && h->eps >= 0.0 && std::isfinite(h->weight_decay),
               "bad rates: lr %g, momentum %g, eps %g, weight decay %g", h->lr, h->momentum, h->eps, h->weight_decay);
    B2_REQUIRE(h->steps >= 1 && h->steps <= kMostSteps && std::isfinite(h->a) && std::isfinite(h->b) && std::isfinite(h->c), "bad polynomial: %d steps of %g, %g, %g",
               h->steps, h->a, h->b, h->c);
    B2_REQUIRE((((uintptr_t)lr | (uintptr_t)grad_scale | (uintptr_t)step | (uintptr_t)status) & 3) == 0, "a number of the step lies between two addresses");
    B2_REQUIRE(!b2::overlap(plan, s->plan_bytes, scratch, s->scratch_bytes), "the plan lies in the scratch");
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
    r.a = (float)h->a;
    r.b = (float)h->b;
    r.c = (float)h->c;
    r.lr = h->lr;
    r.wd = h->weight_decay;
    r.nesterov = h->nesterov != 0;
    cudaStream_t st = (cudaStream_t)stream;
    const void* base = aligned(plan, 64);
    double* sums = (double*)aligned(scratch, 256);
    float* values = (float*)((char*)sums + sums_bytes(s->chunks));
    const long long most = b2::kSms * 8, blocks = s->chunks < 1 ? 1 : s->chunks < most ? s->chunks : most;
    B2_CUDA((b2::launch_after(muon_mean_kernel, dim3((unsigned)blocks), kThreads, 0, st, base, (long long)s->matrices, (long long)s->chunks, (long long)s->items, r,
                              grad_scale, step, sums, values)));
    if (s->items == 0) return B2_OK;
    B2_CUDA((b2::launch_after(muon_scale_kernel, dim3((unsigned)blocks), kThreads, 0, st, base, (long long)s->matrices, (long long)s->chunks, (long long)s->items,
                              r.eps, (const double*)sums, values)));
    for (int k = 0; k < h->steps; ++k)
        for (int phase = 0; phase < 3; ++phase)
            B2_CUDA((b2::launch_after(muon_product_kernel, dim3((unsigned)s->items), kThreads, 0, st, base, (long long)s->matrices, (long long)s->chunks,
                                      (long long)s->items, phase, k & 1, (int)(k == h->steps - 1), r, lr, values)));
    return B2_OK;
}
