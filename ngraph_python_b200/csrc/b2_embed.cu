// Table lookups with a scale and the gradient of the table by sorted tokens.
//
//   forward   out[t, :] = scale * table[token[t], :]
//   gradient  dW[v, :] = scale * sum of delta[t, :] over the t with token[t] = v, t ascending
//
// Both are bound by memory: one multiplication or addition a value.  The gradient is two launches.  The first
// sorts: a CTA owns the rows v = b (mod CTAs), so that the frequent tokens of a vocabulary, which lie next to one
// another, go to different CTAs; it reads every token, counts its own per warp, and writes their positions row by
// row in ascending order, and a list of work items of at most kPart positions each.  No counter is shared between
// CTAs -- where a CTA's positions begin is the number of tokens that lower CTAs own, which it counts as well -- so
// that the order of every sum is that of the tokens, whatever runs when, and nothing has to be cleared in advance.
// The same launch writes the zeros of rows that no token names (all but the sums is bandwidth there).  The second
// adds: a warp takes an item and kCols columns.  Rows of more than kPart positions leave fp32 partial sums, which
// the warp that comes last adds in their order.
#include <cstdint>

#include "b2_operators.h"

namespace {

constexpr int kPart = 32;               // positions in one work item
constexpr int kOrderThreads = 1024;
constexpr int kMostRows = 6400;         // rows that a CTA of the first launch owns, at most
constexpr int kCounters = 50000;        // words of shared memory for their counters

struct FlexArgs {
    const b2_flex_scale* table;
    int slot_in, slot_idx, slot_out;
    int* stats;
    unsigned long long* probe_out;
    int probe;
};

// The token at position i, or -1 where it names no row (also for NaN).
template <int KIND>
__device__ __forceinline__ int token_at(const void* idx, long long i, int V, float step) {
    if (KIND == B2_IDX_F32 || KIND == B2_IDX_FLEX16) {
        const float x = KIND == B2_IDX_F32 ? static_cast<const float*>(idx)[i] : step * (float)static_cast<const short*>(idx)[i];
        const float r = rintf(x);
        return r >= 0.0f && r < (float)V ? (int)r : -1;
    }
    if (KIND == B2_IDX_I32) {
        const int x = static_cast<const int*>(idx)[i];
        return x >= 0 && x < V ? x : -1;
    }
    const long long x = static_cast<const long long*>(idx)[i];
    return x >= 0 && x < V ? (int)x : -1;
}

// V values next to one another, fp32 or mantissas
template <typename T, int VEC> struct Pack;
template <> struct Pack<float, 4> {
    float4 w;
    __device__ __forceinline__ void load(const float* p) { w = *reinterpret_cast<const float4*>(p); }
    __device__ __forceinline__ void get(float* v) const { v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w; }
};
template <> struct Pack<short, 8> {
    int4 w;
    __device__ __forceinline__ void load(const short* p) { w = *reinterpret_cast<const int4*>(p); }
    __device__ __forceinline__ void get(float* v) const {
        const int x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[2 * k] = (float)(short)(x[k] & 0xffff);
            v[2 * k + 1] = (float)(x[k] >> 16);
        }
    }
};
template <typename T> struct Pack<T, 1> {
    T w;
    __device__ __forceinline__ void load(const T* p) { w = *p; }
    __device__ __forceinline__ void get(float* v) const { v[0] = (float)w; }
};

// fp32 to a mantissa, to the nearest even one; `stat` follows the largest
__device__ __forceinline__ int to_mantissa(float v, float& stat) {
    v = v != v ? 0.0f : v;
    v = fminf(fmaxf(v, -32768.0f), 32767.0f);
    stat = fmaxf(stat, fabsf(v));
    return __float_as_int(v + 12582912.0f) - 0x4B400000;
}

// Stores of finished values: fp32 as they are, flex16 with the result's exponent; a measuring launch stores
// nothing and follows the largest value.
template <typename T, int VEC> struct Sink;
template <> struct Sink<float, 4> {
    __device__ __forceinline__ Sink(const FlexArgs&) {}
    __device__ __forceinline__ void put(float* p, const float* v) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
    __device__ __forceinline__ void done(const FlexArgs&) {}
};
template <> struct Sink<float, 1> {
    __device__ __forceinline__ Sink(const FlexArgs&) {}
    __device__ __forceinline__ void put(float* p, const float* v) { *p = v[0]; }
    __device__ __forceinline__ void done(const FlexArgs&) {}
};
template <int VEC> struct Sink<short, VEC> {
    float q, most = 0.0f;
    bool probe;
    __device__ __forceinline__ Sink(const FlexArgs& f) : q(f.probe ? 1.0f : f.table[f.slot_out].inv_scale), probe(f.probe != 0) {}
    __device__ __forceinline__ void put(short* p, const float* v) {
        if (probe) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) most = fmaxf(most, fabsf(v[k]));
            return;
        }
        int m[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) m[k] = to_mantissa(v[k] * q, most);
        if constexpr (VEC == 8) {
            int4 w;
            w.x = (m[0] & 0xffff) | (m[1] << 16);
            w.y = (m[2] & 0xffff) | (m[3] << 16);
            w.z = (m[4] & 0xffff) | (m[5] << 16);
            w.w = (m[6] & 0xffff) | (m[7] << 16);
            *reinterpret_cast<int4*>(p) = w;
        } else {
            *p = (short)m[0];
        }
    }
    // (called by whole warps)
    __device__ __forceinline__ void done(const FlexArgs& f) {
        unsigned bits = probe ? __float_as_uint(most) : (unsigned)(int)rintf(most);
        bits = __reduce_max_sync(0xffffffffu, bits);
        if ((threadIdx.x & 31) == 0 && bits) {
            if (probe) atomicMax(f.probe_out, (unsigned long long)bits);
            else atomicMax(f.stats + f.slot_out, (int)bits);
        }
    }
};

// ---- forward --------------------------------------------------------------------------------------------
// A thread takes UN vectors a block apart: their tokens, then their rows, are loads in flight together.
template <typename T, int VEC, int KIND, int UN>
__global__ void __launch_bounds__(256)
embed_kernel(const T* __restrict__ table, const void* __restrict__ idx, T* __restrict__ out, int V, int F, long long n, float scale, FlexArgs f) {
    after_earlier_kernels();
    const bool flex = sizeof(T) == 2;
    const float step = flex ? f.table[f.slot_in].scale : 1.0f;
    const float istep = KIND == B2_IDX_FLEX16 ? f.table[f.slot_idx].scale : 1.0f;
    Sink<T, VEC> sink(f);
    const unsigned per_row = (unsigned)(F / VEC);
    const long long total = n * per_row;
    for (long long base = (long long)blockIdx.x * (256 * UN) + threadIdx.x; base - threadIdx.x < total; base += (long long)gridDim.x * (256 * UN)) {
        Pack<T, VEC> w[UN];
        int row[UN];
        unsigned col[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const long long e = base + u * 256;
            row[u] = -1;
            col[u] = 0;
            if (e < total) {
                const long long t = total <= 0xffffffffll ? (long long)((unsigned)e / per_row) : e / per_row;
                col[u] = (unsigned)(e - t * per_row) * VEC;
                row[u] = token_at<KIND>(idx, t, V, istep);
            }
        }
#pragma unroll
        for (int u = 0; u < UN; ++u)
            if (row[u] >= 0) w[u].load(table + (long long)row[u] * F + col[u]);
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const long long e = base + u * 256;
            if (e >= total) break;
            float v[VEC] = {};
            if (row[u] >= 0) {
                w[u].get(v);
#pragma unroll
                for (int k = 0; k < VEC; ++k) v[k] = flex ? (v[k] * step) * scale : v[k] * scale;
            }
            sink.put(out + e * VEC, v);
        }
    }
    sink.done(f);
}

// ---- gradient: order ----------------------------------------------------------------------------------------
struct Item {
    int row, first, count, slot;        // slot: where its partial sums go, -1 for a whole row
    int slot0, parts, pad0, pad1;       // of the row
};

struct Scratch {
    int* sorted;                        // [n] positions
    Item* items;                        // [n], those with count 0 are none
    unsigned* tickets;                  // [slots][column blocks]
    float* partial;                     // [slots][F]
    size_t bytes;
};

// 2n / kPart + 2 slots: the ceil(c / kPart) parts of a row of c > kPart positions from `start` on fit between
// 2 start / kPart and 2 (start + c) / kPart, where the next row's begin.
Scratch scratch_of(void* base, int F, long long n, int col_blocks) {
    Scratch s;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        char* p = static_cast<char*>(base) + at;
        at += (bytes + 255) / 256 * 256;
        return p;
    };
    const size_t slots = 2 * (size_t)n / kPart + 2;
    s.items = reinterpret_cast<Item*>(take(n * sizeof(Item)));
    s.sorted = reinterpret_cast<int*>(take(n * sizeof(int)));
    s.tickets = reinterpret_cast<unsigned*>(take(slots * col_blocks * sizeof(unsigned)));
    s.partial = reinterpret_cast<float*>(take(slots * (size_t)F * sizeof(float)));
    s.bytes = at;
    return s;
}

struct OrderArgs {
    const void* idx;
    int V, F, n, rows, warps, pad, col_blocks;
    unsigned magic;                     // 2^32 / CTAs, rounded up
    Scratch s;
    const b2_flex_scale* table;
    int slot_idx;
};

// exclusive sum over the CTA, and the total; `sums` has 33 words
__device__ __forceinline__ unsigned block_scan(unsigned v, unsigned* sums, unsigned& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
        unsigned s = sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        sums[lane] = s;
    }
    __syncthreads();
    total = sums[31];
    return x - v + (warp ? sums[warp - 1] : 0u);
}

template <typename T>
__device__ __forceinline__ void zero_row(T* p, int F, int lane) {
    const int head = min(F, (int)((-(reinterpret_cast<uintptr_t>(p) / sizeof(T))) & (16 / sizeof(T) - 1)));
    if (lane < head) p[lane] = (T)0;
    const int vecs = (F - head) / (int)(16 / sizeof(T));
    for (int i = lane; i < vecs; i += 32) reinterpret_cast<int4*>(p + head)[i] = make_int4(0, 0, 0, 0);
    for (int i = head + vecs * (int)(16 / sizeof(T)) + lane; i < F; i += 32) p[i] = (T)0;
}

// `zeros`: the table of sums, whose rows without tokens become zero here; NULL where sums are added onto it.
template <typename T, int KIND>
__global__ void __launch_bounds__(kOrderThreads)
order_kernel(const OrderArgs a, T* __restrict__ zeros) {
    extern __shared__ unsigned counters[];      // [warps][rows], then [rows] sums
    __shared__ unsigned sums[33];
    after_earlier_kernels();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned G = gridDim.x, b = blockIdx.x;
    const int rows = a.rows;
    unsigned* mine = counters + (size_t)warp * rows;
    unsigned* whole = counters + (size_t)a.warps * rows;
    const float istep = KIND == B2_IDX_FLEX16 ? a.table[a.slot_idx].scale : 1.0f;
    for (int i = threadIdx.x; i < a.warps * rows; i += kOrderThreads) counters[i] = 0;
    __syncthreads();
    // a warp's share of the positions, in whole lines of 32
    const int per = ((a.n + a.warps - 1) / a.warps + 31) / 32 * 32;
    const long long from = (long long)warp * per;
    const int begin = (int)min(from, (long long)a.n), end = warp < a.warps ? (int)min(from + per, (long long)a.n) : begin;

    constexpr int UN = 8;
    // token -> row within the CTA (v / G) and owner (v % G); the estimate of the quotient is at most one too high
    auto split = [&](int v, int& local) {
        unsigned q = __umulhi((unsigned)v, a.magic);
        int r = v - (int)(q * G);
        if (r < 0) { --q; r += (int)G; }
        if (r >= (int)G) { ++q; r -= (int)G; }      // (one CTA: its 2^32 has no word)
        local = (int)q;
        return (unsigned)r;
    };
    unsigned lower = 0;
    for (int at = begin; at < end; at += 32 * UN) {
        int tok[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int i = at + u * 32 + lane;
            tok[u] = i < end ? token_at<KIND>(a.idx, i, a.V, istep) : -1;
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            if (tok[u] < 0 || tok[u] == a.pad) continue;
            int local;
            const unsigned owner = split(tok[u], local);
            if (owner == b) atomicAdd(mine + local, 1u);
            lower += owner < b;
        }
    }
    unsigned start;
    block_scan(lower, sums, start);             // (its barriers also end the counting)
    // counters become where each warp's positions of each row begin; rows' items are listed
    unsigned items = start, begun = start;
    for (int r0 = 0; r0 < rows; r0 += kOrderThreads) {
        const int r = r0 + threadIdx.x;
        unsigned c = 0;
        if (r < rows)
            for (int w = 0; w < a.warps; ++w) {
                const unsigned x = counters[(size_t)w * rows + r];
                counters[(size_t)w * rows + r] = c;
                c += x;
            }
        unsigned all_c, all_p;
        const unsigned first = begun + block_scan(c, sums, all_c);
        const unsigned parts = (c + kPart - 1) / kPart;
        const unsigned item = items + block_scan(parts, sums, all_p);
        if (r < rows) {
            whole[r] = c;
            for (int w = 0; w < a.warps; ++w) counters[(size_t)w * rows + r] += first;
            const int row = (int)(b + (unsigned)r * G);
            const int slot0 = (int)(2ull * first / kPart);
            for (unsigned p = 0; p < parts; ++p) {
                Item it;
                it.row = row;
                it.first = (int)(first + p * kPart);
                it.count = (int)min((unsigned)kPart, c - p * kPart);
                it.slot = parts > 1 ? slot0 + (int)p : -1;
                it.slot0 = slot0;
                it.parts = (int)parts;
                it.pad0 = it.pad1 = 0;
                a.s.items[item + p] = it;
            }
            if (parts > 1)
                for (int k = 0; k < a.col_blocks; ++k) a.s.tickets[(size_t)slot0 * a.col_blocks + k] = 0;
        }
        begun += all_c;
        items += all_p;
    }
    // items that are none: up to where the next CTA's begin, the last CTA's up to n
    const unsigned last = b + 1 == G ? (unsigned)a.n : begun;
    for (unsigned i = items + threadIdx.x; i < last; i += kOrderThreads) a.s.items[i].count = 0;
    __syncthreads();
    if (zeros)
        for (int r = warp; r < rows; r += kOrderThreads / 32) {
            const long long row = (long long)b + (long long)r * G;
            if (row < a.V && whole[r] == 0) zero_row(zeros + row * a.F, a.F, lane);
        }
    // positions, in the order of the tokens
    for (int at = begin; at < end; at += 32 * UN) {
        int tok[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int i = at + u * 32 + lane;
            tok[u] = i < end ? token_at<KIND>(a.idx, i, a.V, istep) : -1;
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            int local = 0;
            const bool ours = tok[u] >= 0 && tok[u] != a.pad && split(tok[u], local) == b;
            const unsigned those = __ballot_sync(0xffffffffu, ours);
            if (!those) continue;
            if (ours) {
                const unsigned same = __match_any_sync(those, local);
                const unsigned before = mine[local];
                __syncwarp(those);
                const int rank = __popc(same & ((1u << lane) - 1u));
                a.s.sorted[before + rank] = at + u * 32 + lane;
                if (rank == 0) mine[local] = before + __popc(same);
            }
            __syncwarp();
        }
    }
}

// ---- gradient: sums -------------------------------------------------------------------------------------------
// Partial sums go past the first cache, which another SM's stores do not reach.
template <int VEC>
__device__ __forceinline__ void put_sums(float* p, const float* v) {
    if constexpr (VEC % 4 == 0) {
#pragma unroll
        for (int k = 0; k < VEC; k += 4) __stcg(reinterpret_cast<float4*>(p + k), make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]));
    } else {
        __stcg(p, v[0]);
    }
}
template <int VEC>
__device__ __forceinline__ void add_sums(const float* p, float* v) {
    if constexpr (VEC % 4 == 0) {
#pragma unroll
        for (int k = 0; k < VEC; k += 4) {
            const float4 w = __ldcg(reinterpret_cast<const float4*>(p + k));
            v[k] += w.x; v[k + 1] += w.y; v[k + 2] += w.z; v[k + 3] += w.w;
        }
    } else {
        v[0] += __ldcg(p);
    }
}

// A warp takes an item and 32 * VEC * UN columns.
template <typename T, int VEC, int UN>
__global__ void __launch_bounds__(256)
sum_kernel(const T* __restrict__ delta, T* __restrict__ dW, int F, int n, float scale, int onto, int col_blocks, Scratch s, FlexArgs f) {
    after_earlier_kernels();
    constexpr int COLS = 32 * VEC;
    const bool flex = sizeof(T) == 2;
    const float step = flex ? f.table[f.slot_in].scale : 1.0f;
    Sink<T, VEC> sink(f);
    const int lane = threadIdx.x & 31;
    const long long units = (long long)n * col_blocks;
    for (long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); unit < units; unit += (long long)gridDim.x * 8) {
        const int which = (int)(unit / col_blocks), block = (int)(unit - (long long)which * col_blocks);
        const int4 it = *reinterpret_cast<const int4*>(s.items + which);
        const int row = it.x, first = it.y, count = it.z, slot = it.w;
        if (count == 0) continue;
        const int col0 = block * COLS * UN + lane * VEC;
        float acc[UN][VEC] = {};
        const int at = lane < count ? s.sorted[first + lane] : 0;
        constexpr int AHEAD = 4;
        for (int j = 0; j < count; j += AHEAD) {
            Pack<T, VEC> w[AHEAD][UN];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const long long t = __shfl_sync(0xffffffffu, at, (j + a) & 31);
#pragma unroll
                for (int u = 0; u < UN; ++u)
                    if (j + a < count && col0 + u * COLS < F) w[a][u].load(delta + t * F + col0 + u * COLS);
            }
#pragma unroll
            for (int a = 0; a < AHEAD; ++a)
#pragma unroll
                for (int u = 0; u < UN; ++u)
                    if (j + a < count && col0 + u * COLS < F) {
                        float v[VEC];
                        w[a][u].get(v);
#pragma unroll
                        for (int k = 0; k < VEC; ++k) acc[u][k] += v[k];
                    }
        }
        if (slot >= 0) {
            const int4 more = reinterpret_cast<const int4*>(s.items + which)[1];
            const int slot0 = more.x, parts = more.y;
#pragma unroll
            for (int u = 0; u < UN; ++u)
                if (col0 + u * COLS < F) put_sums<VEC>(s.partial + (long long)slot * F + col0 + u * COLS, acc[u]);
            __threadfence();
            __syncwarp();
            unsigned came = 0;
            if (lane == 0) came = atomicAdd(s.tickets + (long long)slot0 * col_blocks + block, 1u);
            came = __shfl_sync(0xffffffffu, came, 0);
            if (came + 1 != (unsigned)parts) continue;
            __threadfence();
#pragma unroll
            for (int u = 0; u < UN; ++u)
#pragma unroll
                for (int k = 0; k < VEC; ++k) acc[u][k] = 0.0f;
            for (int p = 0; p < parts; ++p)
#pragma unroll
                for (int u = 0; u < UN; ++u)
                    if (col0 + u * COLS < F) add_sums<VEC>(s.partial + (long long)(slot0 + p) * F + col0 + u * COLS, acc[u]);
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int col = col0 + u * COLS;
            if (col >= F) break;
            T* p = dW + (long long)row * F + col;
            float v[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[k] = flex ? (acc[u][k] * step) * scale : acc[u][k] * scale;
            if (!flex && onto) {
                Pack<T, VEC> old;
                old.load(p);
                float o[VEC];
                old.get(o);
#pragma unroll
                for (int k = 0; k < VEC; ++k) v[k] = o[k] + v[k];
            }
            sink.put(p, v);
        }
    }
    sink.done(f);
}

// columns of a warp of sum_kernel in vectors of VEC
constexpr int kUn = 2;
int col_blocks_of(int F, int vec) { return (F + 32 * vec * kUn - 1) / (32 * vec * kUn); }

template <typename T> constexpr int wide() { return 16 / (int)sizeof(T); }

template <typename T, int KIND>
int launch_embed(const void* table, const void* idx, void* out, int V, int F, long long n, float scale, const FlexArgs& f, cudaStream_t st) {
    constexpr int W = wide<T>();
    const bool vec = F % W == 0 && b2::aligned16(table) && b2::aligned16(out);
    const long long total = n * (long long)(vec ? F / W : F);
    // four vectors a thread hide the two loads behind one another; where that leaves SMs without a block, one
    const bool deep = total >= 4ll * 256 * b2::kSms;
    long long blocks = (total + (deep ? 1023 : 255)) / (deep ? 1024 : 256);
    if (blocks > (1ll << 30)) blocks = 1ll << 30;
#define B2_EMBED(VEC, UN) \
    B2_CUDA((b2::launch_after(embed_kernel<T, VEC, KIND, UN>, dim3((unsigned)blocks), 256, 0, st, (const T*)table, idx, (T*)out, V, F, n, scale, f)))
    if (vec && deep) B2_EMBED(W, 4);
    else if (vec) B2_EMBED(W, 1);
    else if (deep) B2_EMBED(1, 4);
    else B2_EMBED(1, 1);
#undef B2_EMBED
    return B2_OK;
}

template <typename T, int KIND>
int launch_order(OrderArgs a, T* zeros, cudaStream_t st) {
    static std::atomic<unsigned long long> done{0};
    B2_CHECK(b2::allow_shared((const void*)order_kernel<T, KIND>, (kCounters + kMostRows) * 4, &done));
    int ctas = a.V < b2::kSms ? a.V : b2::kSms;
    const int least = (int)(((long long)a.V + kMostRows - 1) / kMostRows);
    if (ctas < least) ctas = least;
    a.rows = (a.V + ctas - 1) / ctas;
    a.magic = ctas == 1 ? 0xffffffffu : (unsigned)((1ull << 32) / ctas + 1);
    a.warps = kCounters / a.rows - 1;
    if (a.warps > kOrderThreads / 32) a.warps = kOrderThreads / 32;
    const size_t smem = (size_t)(a.warps + 1) * a.rows * 4;
    B2_CUDA((b2::launch_after(order_kernel<T, KIND>, dim3((unsigned)ctas), kOrderThreads, smem, st, a, zeros)));
    return B2_OK;
}

template <typename T>
int launch_update(const void* delta, const void* idx, void* dW, int kind, int V, int F, long long n, float scale, int pad, int onto, const FlexArgs& f,
                  void* scratch, cudaStream_t st) {
    constexpr int W = wide<T>();
    const bool vec = F % W == 0 && b2::aligned16(delta) && b2::aligned16(dW);
    OrderArgs a;
    a.idx = idx;
    a.V = V;
    a.F = F;
    a.n = (int)n;
    a.pad = pad;
    a.col_blocks = col_blocks_of(F, vec ? W : 1);
    a.s = scratch_of(scratch, F, n, a.col_blocks);
    a.table = f.table;
    a.slot_idx = f.slot_idx;
    T* zeros = onto || f.probe ? nullptr : (T*)dW;
    if (kind == B2_IDX_F32) B2_CHECK((launch_order<T, B2_IDX_F32>(a, zeros, st)));
    else if (kind == B2_IDX_I32) B2_CHECK((launch_order<T, B2_IDX_I32>(a, zeros, st)));
    else if (kind == B2_IDX_I64) B2_CHECK((launch_order<T, B2_IDX_I64>(a, zeros, st)));
    else B2_CHECK((launch_order<T, B2_IDX_FLEX16>(a, zeros, st)));
    if (n == 0) return B2_OK;
    long long blocks = (n * a.col_blocks + 7) / 8;
    if (blocks > b2::kSms * 8) blocks = b2::kSms * 8;
    if (vec)
        B2_CUDA((b2::launch_after(sum_kernel<T, W, kUn>, dim3((unsigned)blocks), 256, 0, st, (const T*)delta, (T*)dW, F, (int)n, scale, onto, a.col_blocks, a.s, f)));
    else
        B2_CUDA((b2::launch_after(sum_kernel<T, 1, kUn>, dim3((unsigned)blocks), 256, 0, st, (const T*)delta, (T*)dW, F, (int)n, scale, onto, a.col_blocks, a.s, f)));
    return B2_OK;
}

int check_flex(int flex, int kind, const FlexArgs& f) {
    B2_REQUIRE(kind >= B2_IDX_F32 && kind <= B2_IDX_FLEX16, "unknown kind of index: %d", kind);
    B2_REQUIRE(kind != B2_IDX_FLEX16 || (f.table && f.slot_idx >= 0), "a flex16 index needs the scale table");
    if (!flex) return B2_OK;
    B2_REQUIRE(f.table && f.slot_in >= 0 && f.slot_out >= 0, "a flex16 lookup needs the scale table");
    B2_REQUIRE(f.probe ? f.probe_out != nullptr : f.stats != nullptr, "missing statistics destination");
    return B2_OK;
}

}  // namespace

extern "C" int b2_embed_fprop(const void* table, const void* idx, void* out, int32_t flex, int32_t idx_kind, int32_t V, int32_t F, int64_t n_idx,
                              float scale, const b2_flex_scale* scales, int32_t slot_table, int32_t slot_idx, int32_t slot_out, int32_t* stats,
                              uint64_t* probe_out, int32_t probe, void* stream) {
    B2_REQUIRE(V > 0 && F > 0 && n_idx >= 0, "bad lookup: table %d x %d, %lld tokens", V, F, (long long)n_idx);
    const FlexArgs f = {scales, slot_table, slot_idx, slot_out, stats, (unsigned long long*)probe_out, probe ? 1 : 0};
    B2_CHECK(check_flex(flex, idx_kind, f));
    if (n_idx == 0) return B2_OK;
    B2_REQUIRE(table && idx && out, "bad lookup: missing tensor");
    B2_CHECK(b2::require_here(out, "the lookup's result"));
    cudaStream_t st = (cudaStream_t)stream;
#define B2_KIND(T)                                                                                                          \
    switch (idx_kind) {                                                                                                     \
        case B2_IDX_F32: return launch_embed<T, B2_IDX_F32>(table, idx, out, V, F, n_idx, scale, f, st);                    \
        case B2_IDX_I32: return launch_embed<T, B2_IDX_I32>(table, idx, out, V, F, n_idx, scale, f, st);                    \
        case B2_IDX_I64: return launch_embed<T, B2_IDX_I64>(table, idx, out, V, F, n_idx, scale, f, st);                    \
        default: return launch_embed<T, B2_IDX_FLEX16>(table, idx, out, V, F, n_idx, scale, f, st);                         \
    }
    if (flex) B2_KIND(short)
    B2_KIND(float)
#undef B2_KIND
}

extern "C" int b2_embed_update_scratch_bytes(int32_t V, int32_t F, int64_t n_idx, size_t* bytes) {
    B2_REQUIRE(bytes && V > 0 && F > 0 && n_idx >= 0 && n_idx <= (1ll << 30), "bad lookup: table %d x %d, %lld tokens", V, F, (long long)n_idx);
    *bytes = scratch_of(nullptr, F, n_idx, col_blocks_of(F, 1)).bytes + 256;
    return B2_OK;
}

extern "C" int b2_embed_update(const void* delta, const void* idx, void* dW, int32_t flex, int32_t idx_kind, int32_t V, int32_t F, int64_t n_idx,
                               float scale, int64_t pad_idx, int32_t onto, const b2_flex_scale* scales, int32_t slot_delta, int32_t slot_idx,
                               int32_t slot_dW, int32_t* stats, uint64_t* probe_out, int32_t probe, void* scratch, size_t scratch_bytes, void* stream) {
    size_t need = 0;
    B2_CHECK(b2_embed_update_scratch_bytes(V, F, n_idx, &need));
    const FlexArgs f = {scales, slot_delta, slot_idx, slot_dW, stats, (unsigned long long*)probe_out, probe ? 1 : 0};
    B2_CHECK(check_flex(flex, idx_kind, f));
    B2_REQUIRE(!(flex && onto), "flex16 sums have an exponent of their own: they are not added onto a table");
    B2_REQUIRE(dW && (n_idx == 0 || (delta && idx)), "bad lookup gradient: missing tensor");
    B2_REQUIRE(scratch && scratch_bytes >= need, "the lookup's gradient needs %zu bytes of scratch, got %zu", need, scratch_bytes);
    B2_CHECK(b2::require_here(dW, "the table's gradient"));
    const int pad = pad_idx >= 0 && pad_idx < V ? (int)pad_idx : -1;
    void* at = (void*)(((uintptr_t)scratch + 255) / 256 * 256);
    if (flex) return launch_update<short>(delta, idx, dW, idx_kind, V, F, n_idx, scale, pad, onto, f, at, (cudaStream_t)stream);
    return launch_update<float>(delta, idx, dW, idx_kind, V, F, n_idx, scale, pad, onto ? 1 : 0, f, at, (cudaStream_t)stream);
}
