// Table lookups with a scale and the gradient of the table by sorted tokens.
//
//   forward   out[t, :] = scale * table[token[t], :]
//   gradient  dW[v, :] = scale * sum of delta[t, :] over the t with token[t] = v, t ascending
//
// Both are bound by memory: one multiplication or addition a value (16384 x 1024 looked up: 17.8 us, 0.77 of the rate of a
// copy; 8192 x 1024 added into 32000 rows: 32.5 us, of which the sort takes 7 and 18 are zeros).  The gradient is two launches.  The first
// sorts: a CTA owns the rows v = b (mod CTAs), so that the frequent tokens of a vocabulary, which lie next to one
// another, go to different CTAs; it reads every token, counts its own per warp, and writes their positions row by
// row in ascending order.  No counter is shared between CTAs -- where a CTA's positions begin is the number of tokens
// that lower CTAs own, which it counts as well -- so that the order of every sum is that of the tokens, whatever runs
// when, and nothing has to be cleared in advance.  The second adds, in parts of at most kPart positions of a row; rows
// of more leave fp32 partial sums, which the warp that comes last adds in their order.
#include <cstdint>
#include <type_traits>

#include "b2_operators.h"

namespace {

constexpr int kPart = 32;               // positions in one work item
constexpr int kOrderThreads = 1024;
constexpr int kMostRows = 4000;         // rows that a CTA of the first launch owns, at most
constexpr int kCounters = 25000;        // words of shared memory for them
constexpr int kListed = 128;            // own tokens that a warp remembers
constexpr int kFlat = 2048;             // ... and a CTA

struct FlexArgs {
    const b2_flex_scale* table;
    int slot_in, slot_idx, slot_out;
    int* stats;
    unsigned long long* probe_out;
    int probe;
};

// How tokens of a kind are held, and the row that one names: -1 for none (also for NaN).  fp32 to the nearest row.
template <int KIND> struct Held { using Type = float; };
template <> struct Held<B2_IDX_I32> { using Type = int; };
template <> struct Held<B2_IDX_I64> { using Type = long long; };
template <> struct Held<B2_IDX_FLEX16> { using Type = short; };

__device__ __forceinline__ int row_of(float x, int V, float) {
    const int r = __float2int_rn(x);
    return (unsigned)r < (unsigned)V && x == x ? r : -1;
}
__device__ __forceinline__ int row_of(int x, int V, float) { return (unsigned)x < (unsigned)V ? x : -1; }
__device__ __forceinline__ int row_of(long long x, int V, float) { return (unsigned long long)x < (unsigned long long)V ? (int)x : -1; }
__device__ __forceinline__ int row_of(short x, int V, float step) { return row_of(step * (float)x, V, 0.0f); }

template <int KIND>
__device__ __forceinline__ int token_at(const void* idx, long long i, int V, float step) {
    return row_of(static_cast<const typename Held<KIND>::Type*>(idx)[i], V, step);
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
template <> struct Pack<short, 4> {
    int2 w;
    __device__ __forceinline__ void load(const short* p) { w = *reinterpret_cast<const int2*>(p); }
    __device__ __forceinline__ void get(float* v) const {
        v[0] = (float)(short)(w.x & 0xffff);
        v[1] = (float)(w.x >> 16);
        v[2] = (float)(short)(w.y & 0xffff);
        v[3] = (float)(w.y >> 16);
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
        } else if constexpr (VEC == 4) {
            *reinterpret_cast<int2*>(p) = make_int2((m[0] & 0xffff) | (m[1] << 16), (m[2] & 0xffff) | (m[3] << 16));
        } else {
            *p = (short)m[0];
        }
    }
    // (called by whole warps)
    __device__ __forceinline__ void done(const FlexArgs& f) {
        unsigned bits = probe ? __float_as_uint(most) : (unsigned)(int)rintf(most);
        bits = __reduce_max_sync(0xffffffffu, bits);
        if ((threadIdx.x & 31) != 0) return;
        // (an atomic only where it would change the word: thousands of warps come with nothing new)
        if (probe) {
            if (bits > __ldcg(f.probe_out)) atomicMax(f.probe_out, (unsigned long long)bits);
        } else if ((int)bits > __ldcg(f.stats + f.slot_out)) {
            atomicMax(f.stats + f.slot_out, (int)bits);
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

// Rows that are not aligned: a warp takes 32 * UN columns of a token.  (In the order of the result's values, with a
// division for each, 16384 x 1001 took 38 us, flex16 89.)
template <typename T, int KIND, int UN>
__global__ void __launch_bounds__(256)
embed_apart_kernel(const T* __restrict__ table, const void* __restrict__ idx, T* __restrict__ out, int V, int F, long long n, unsigned col_blocks, float scale,
                   FlexArgs f) {
    after_earlier_kernels();
    const bool flex = sizeof(T) == 2;
    const float step = flex ? f.table[f.slot_in].scale : 1.0f;
    const float istep = KIND == B2_IDX_FLEX16 ? f.table[f.slot_idx].scale : 1.0f;
    Sink<T, 1> sink(f);
    const long long units = n * col_blocks;
    for (long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); unit < units; unit += (long long)gridDim.x * 8) {
        const long long t = units <= 0xffffffffll ? (long long)((unsigned)unit / col_blocks) : unit / col_blocks;
        const int col = (int)(unit - t * col_blocks) * 32 * UN + (int)(threadIdx.x & 31);
        const int row = token_at<KIND>(idx, t, V, istep);
        const T* from = table + (long long)(row < 0 ? 0 : row) * F + col;
        T* to = out + t * F + col;
        T w[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u)
            if (col + u * 32 < F) w[u] = from[u * 32];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            if (col + u * 32 >= F) break;
            float v = row < 0 ? 0.0f : (float)w[u];
            v = flex ? (v * step) * scale : v * scale;
            if (row < 0) v = 0.0f;
            sink.put(to + u * 32, &v);
        }
    }
    sink.done(f);
}

// ---- gradient: order ----------------------------------------------------------------------------------------
// A position in the sorted list: of `count` positions of its row it is number `rank`.  row -1: none.
struct Entry {
    int pos, row, rank, count;
};

struct Scratch {
    Entry* sorted;                      // [n]
    unsigned char* used;                // [CTAs][rows of one]: whether a token names the row
    unsigned* tickets;                  // [slots][column blocks]
    float* partial;                     // [slots][F]
    size_t bytes;
};

// CTAs of the first launch, and rows that each owns
int owners_of(int V) {
    const int least = (int)(((long long)V + kMostRows - 1) / kMostRows);
    const int most = V < b2::kSms ? V : b2::kSms;
    return most > least ? most : least;
}

// 2n / kPart + 2 slots: the ceil(c / kPart) parts of a row of c > kPart positions from `start` on fit between
// 2 start / kPart and 2 (start + c) / kPart, where the next row's begin.
Scratch scratch_of(void* base, int V, int F, long long n, int col_blocks) {
    Scratch s;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        char* p = static_cast<char*>(base) + at;
        at += (bytes + 255) / 256 * 256;
        return p;
    };
    const size_t slots = 2 * (size_t)n / kPart + 2;
    s.sorted = reinterpret_cast<Entry*>(take(n * sizeof(Entry)));
    s.used = reinterpret_cast<unsigned char*>(take((size_t)V + owners_of(V)));
    s.tickets = reinterpret_cast<unsigned*>(take(slots * col_blocks * sizeof(unsigned)));
    s.partial = reinterpret_cast<float*>(take(slots * (size_t)F * sizeof(float)));
    s.bytes = at;
    return s;
}

struct OrderArgs {
    const void* idx;
    int V, n, rows, warps, stride, pad, col_blocks;
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

// A CTA remembers its own tokens in the order of their positions (every warp a list, then one list of all).  One warp
// goes through that, 32 at a time, and numbers the positions of each row; rows get their places in the order in which
// they come up.  A CTA of more than kFlat tokens reads all tokens again: it counts rows per warp, and then places.
template <int KIND>
__global__ void __launch_bounds__(kOrderThreads)
order_kernel(const OrderArgs a) {
    extern __shared__ __align__(16) unsigned room[];
    __shared__ unsigned sums[33], found_by[32];
    constexpr int WARPS = kOrderThreads / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned G = gridDim.x, b = blockIdx.x;
    const int rows = a.rows;
    unsigned* whole = room;                     // [rows] positions of each row, then [rows] where they begin
    unsigned* first = room + rows;
    uint2* lists = reinterpret_cast<uint2*>(room + (2 * rows + 3) / 4 * 4);     // [WARPS][kListed] position and row
    uint2* flat = lists + WARPS * kListed;
    unsigned* ranks = reinterpret_cast<unsigned*>(flat + kFlat);
    for (int i = threadIdx.x; i < rows; i += kOrderThreads) whole[i] = 0;
    after_earlier_kernels();
    const float istep = KIND == B2_IDX_FLEX16 ? a.table[a.slot_idx].scale : 1.0f;

    // the tokens of a warp's share of the positions, 32 at a time: visit(owner, row of the owner, position), by whole
    // warps; owner G for none
    auto tokens = [&](int warps, auto visit) {
        using Type = typename Held<KIND>::Type;
        constexpr int UN = 8;
        const int per = ((a.n + warps - 1) / warps + 31) / 32 * 32;
        const long long from = (long long)warp * per;
        const int begin = (int)min(from, (long long)a.n), end = warp < warps ? (int)min(from + per, (long long)a.n) : begin;
        const Type* list = static_cast<const Type*>(a.idx) + lane;
        for (int at = begin; at < end; at += 32 * UN) {
            Type x[UN];
            const bool whole = at + 32 * UN <= end;
            if (whole) {
#pragma unroll
                for (int u = 0; u < UN; ++u) x[u] = list[at + u * 32];
            } else {
#pragma unroll
                for (int u = 0; u < UN; ++u) x[u] = at + u * 32 + lane < end ? list[at + u * 32] : (Type)0;
            }
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const int v = whole || at + u * 32 + lane < end ? row_of(x[u], a.V, istep) : -1;
                // v / G, at most one too high, and v % G
                unsigned q = __umulhi((unsigned)v, a.magic);
                int r = v - (int)(q * G);
                if (r < 0) { --q; r += (int)G; }
                visit(v >= 0 && v != a.pad ? (unsigned)r : G, (int)q, at + u * 32 + lane);
            }
        }
    };
    unsigned lower = 0, found = 0;
    tokens(WARPS, [&](unsigned owner, int local, int pos) {
        lower += owner < b;
        const unsigned those = __ballot_sync(0xffffffffu, owner == b);
        if (!those) return;
        const unsigned k = found + __popc(those & ((1u << lane) - 1u));
        if (owner == b && k < kListed) lists[warp * kListed + k] = make_uint2((unsigned)pos, (unsigned)local);
        found += __popc(those);
    });
    if (lane == 0) found_by[warp] = found;
    unsigned start;
    block_scan(lower, sums, start);             // (its barriers stand behind the lists, too)
    unsigned before = 0, all = 0, most = 0;
    {
        const unsigned c = found_by[lane];
        all = __reduce_add_sync(0xffffffffu, c);
        most = __reduce_max_sync(0xffffffffu, c);
        before = __reduce_add_sync(0xffffffffu, lane < warp ? c : 0u);
    }
    auto begin_row = [&](unsigned c, unsigned at) {
        if (c > kPart)
            for (int k = 0; k < a.col_blocks; ++k) a.s.tickets[(size_t)(2ull * at / kPart) * a.col_blocks + k] = 0;
    };
    auto put_entry = [&](unsigned pos, unsigned local, unsigned rank) {
        *reinterpret_cast<int4*>(a.s.sorted + first[local] + rank) = make_int4((int)pos, (int)(b + local * G), (int)rank, (int)whole[local]);
    };
    if (most <= kListed && all <= kFlat) {
        for (unsigned k = lane; k < found; k += 32) flat[before + k] = lists[warp * kListed + k];
        __syncthreads();
        if (warp == 0)
            for (unsigned k = lane; k - lane < all; k += 32) {
                const unsigned mine = k < all ? flat[k].y : 0xffffffffu;
                const unsigned same = __match_any_sync(0xffffffffu, mine);
                const unsigned c = k < all ? whole[mine] : 0u, place = __popc(same & ((1u << lane) - 1u));
                __syncwarp();
                if (k < all) {
                    ranks[k] = c + place;
                    if (place == 0) whole[mine] = c + __popc(same);
                }
                __syncwarp();
            }
        __syncthreads();
        unsigned at = start;
        for (unsigned k0 = 0; k0 < all; k0 += kOrderThreads) {
            const unsigned k = k0 + threadIdx.x;
            const unsigned c = k < all && ranks[k] == 0 ? whole[flat[k].y] : 0u;
            unsigned total;
            const unsigned mine = at + block_scan(c, sums, total);
            if (c) {
                first[flat[k].y] = mine;
                begin_row(c, mine);
            }
            at += total;
        }
        start = at;
        __syncthreads();
        for (unsigned k = threadIdx.x; k < all; k += kOrderThreads) put_entry(flat[k].x, flat[k].y, ranks[k]);
    } else {
        unsigned* counters = room + 2 * rows;   // [rows][stride], a word for each warp
        for (int i = threadIdx.x; i < rows * a.stride; i += kOrderThreads) counters[i] = 0;
        __syncthreads();
        tokens(a.warps, [&](unsigned owner, int local, int) {
            if (owner == b) atomicAdd(counters + (size_t)local * a.stride + warp, 1u);
        });
        __syncthreads();
        // a row's counters become where each warp's positions begin among the row's
        for (int r = warp; r < rows; r += WARPS) {
            unsigned* c = counters + (size_t)r * a.stride;
            const unsigned v = lane < a.warps ? c[lane] : 0u;
            unsigned x = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            if (lane < a.warps) c[lane] = x - v;
            if (lane == 31) whole[r] = x;
        }
        __syncthreads();
        for (int r0 = 0; r0 < rows; r0 += kOrderThreads) {
            const int r = r0 + threadIdx.x;
            const unsigned c = r < rows ? whole[r] : 0u;
            unsigned total;
            const unsigned mine = start + block_scan(c, sums, total);
            if (r < rows) {
                first[r] = mine;
                begin_row(c, mine);
            }
            start += total;
        }
        __syncthreads();
        tokens(a.warps, [&](unsigned owner, int local, int pos) {
            const unsigned those = __ballot_sync(0xffffffffu, owner == b);
            if (!those) return;
            if (owner == b) {
                unsigned* c = counters + (size_t)local * a.stride + warp;
                const unsigned same = __match_any_sync(those, local);
                const unsigned rank = *c, place = __popc(same & ((1u << lane) - 1u));
                __syncwarp(those);
                put_entry((unsigned)pos, (unsigned)local, rank + place);
                if (place == 0) *c = rank + __popc(same);
            }
            __syncwarp();
        });
    }
    for (int r = threadIdx.x; r < rows; r += kOrderThreads) a.s.used[(size_t)b * rows + r] = whole[r] != 0;
    if (b + 1 == G)                             // what is left is nobody's: tokens that name no row, or pad
        for (unsigned i = start + threadIdx.x; i < (unsigned)a.n; i += kOrderThreads) a.s.sorted[i].row = -1;
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
__device__ __forceinline__ void get_sums(const float* p, float* v) {
    if constexpr (VEC % 4 == 0) {
#pragma unroll
        for (int k = 0; k < VEC; k += 4) {
            const float4 w = __ldcg(reinterpret_cast<const float4*>(p + k));
            v[k] = w.x; v[k + 1] = w.y; v[k + 2] = w.z; v[k + 3] = w.w;
        }
    } else {
        v[0] = __ldcg(p);
    }
}

template <typename T>
__device__ __forceinline__ void zero_row(T* p, int F, int lane) {
    const int head = min(F, (int)((-(reinterpret_cast<uintptr_t>(p) / sizeof(T))) & (16 / sizeof(T) - 1)));
    if (lane < head) p[lane] = (T)0;
    const int vecs = (F - head) / (int)(16 / sizeof(T));
    for (int i = lane; i < vecs; i += 32) reinterpret_cast<int4*>(p + head)[i] = make_int4(0, 0, 0, 0);
    for (int i = head + vecs * (int)(16 / sizeof(T)) + lane; i < F; i += 32) p[i] = (T)0;
}

struct SumArgs {
    int V, F, n, rows, owners, zero_rows;      // rows without tokens are looked for among zero_rows by a warp
    unsigned col_blocks, sum_blocks;
    float scale;
    Scratch s;
};

// A warp takes the parts that begin among WINDOW places of the sorted list, and 32 * VEC * UN columns: first the
// tokens of these places, loaded together whatever rows they belong to, then what the last part has beyond them, eight
// at a time.  So a thousand tokens that occur once cost little more than one that occurs a thousand times.  The blocks
// behind the first sum_blocks write the zeros of rows that no token names.  Blocks of four warps: where a row has many
// tokens one warp of eight has a part to add and the others' places wait for it (16384 x 1024 into 300 rows 36 us a call
// with eight, 30 with four, 32 with two; 16384 x 768 onto 50000 32, 27 and 28).
constexpr int kSumWarps = 4;

template <typename T, int VEC, int UN, int WINDOW, bool ONTO>
__global__ void __launch_bounds__(32 * kSumWarps)
sum_kernel(const T* __restrict__ delta, T* dW, const SumArgs a, const FlexArgs f) {
    after_earlier_kernels();
    constexpr int COLS = 32 * VEC;
    constexpr bool flex = sizeof(T) == 2;
    // Of mantissas a part's sum is a whole number of at most 2^20, which fp32 holds.  That of 2^30 tokens is not: the parts
    // are added as integers, and rounded once.
    using Sum = typename std::conditional<flex, long long, float>::type;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (blockIdx.x >= a.sum_blocks) {
        const long long from = ((long long)(blockIdx.x - a.sum_blocks) * kSumWarps + warp) * a.zero_rows, mine = from + lane;
        const bool empty = lane < a.zero_rows && mine < (long long)a.owners * a.rows && !a.s.used[mine];
        for (unsigned left = __ballot_sync(0xffffffffu, empty); left; left &= left - 1) {
            const unsigned k = (unsigned)(from + __ffs(left) - 1);
            const long long row = k / (unsigned)a.rows + (long long)(k % (unsigned)a.rows) * a.owners;
            if (row < a.V) zero_row(dW + row * a.F, a.F, lane);
        }
        return;
    }
    const int F = a.F, block = blockIdx.x % a.col_blocks;
    const float step = flex ? f.table[f.slot_in].scale : 1.0f;
    Sink<T, VEC> sink(f);
    const int base = (int)(blockIdx.x / a.col_blocks * kSumWarps + warp) * WINDOW;
    // entries of this window and of what a part that begins in it can reach
    const int4 none = make_int4(0, -1, 0, 0);
    const int4* list = reinterpret_cast<const int4*>(a.s.sorted);
    const int4 near = base + lane < a.n ? list[base + lane] : none;
    const int far = lane < WINDOW && base + 32 + lane < a.n ? list[base + 32 + lane].x : 0;
    // parts begin where the rank is a multiple of kPart; the last of this window ends where its row or its 32 do
    const unsigned those = __ballot_sync(0xffffffffu, lane < WINDOW && near.y >= 0 && near.z % kPart == 0);
    if (those) {
        const int from = __ffs(those) - 1, last = 31 - __clz(those);
        const int upto = last + __shfl_sync(0xffffffffu, min(kPart, near.w - near.z), last);
        const int col0 = block * COLS * UN + lane * VEC;
        float acc[UN][VEC] = {};
        int join_row[2] = {-1, -1}, join_slot[2], join_parts[2];
        auto store = [&](int row, const Pack<T, VEC>* old) {
            T* p = dW + (long long)row * F + col0;
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                if (col0 + u * COLS >= F) continue;
                float v[VEC];
#pragma unroll
                for (int c = 0; c < VEC; ++c) v[c] = flex ? (acc[u][c] * step) * a.scale : acc[u][c] * a.scale;
                if constexpr (ONTO) {
                    float o[VEC];
                    old[u].get(o);
#pragma unroll
                    for (int c = 0; c < VEC; ++c) v[c] = o[c] + v[c];
                }
                sink.put(p + u * COLS, v);
            }
        };
        auto load = [&](const T* from_row, Pack<T, VEC>* w) {
#pragma unroll
            for (int u = 0; u < UN; ++u)
                if (col0 + u * COLS < F) w[u].load(from_row + col0 + u * COLS);
        };
        auto add = [&](const Pack<T, VEC>* w) {
#pragma unroll
            for (int u = 0; u < UN; ++u)
                if (col0 + u * COLS < F) {
                    float v[VEC];
                    w[u].get(v);
#pragma unroll
                    for (int c = 0; c < VEC; ++c) acc[u][c] += v[c];
                }
        };
        // a part of a row of several ends: `at` is its last place
        auto leave = [&](int which, int at, int row, int rank, int count) {
            join_row[which] = row;
            join_slot[which] = (int)(2ll * (base + at - rank) / kPart);
            join_parts[which] = (count + kPart - 1) / kPart;
#pragma unroll
            for (int u = 0; u < UN; ++u)
                if (col0 + u * COLS < F) put_sums<VEC>(a.s.partial + (long long)(join_slot[which] + rank / kPart) * F + col0 + u * COLS, acc[u]);
        };
        Pack<T, VEC> w[WINDOW][UN], old[ONTO ? WINDOW : 1][UN];
#pragma unroll
        for (int k = 0; k < WINDOW; ++k) {
            const long long t = __shfl_sync(0xffffffffu, near.x, k);
            const int row = __shfl_sync(0xffffffffu, near.y, k), rank = __shfl_sync(0xffffffffu, near.z, k), count = __shfl_sync(0xffffffffu, near.w, k);
            if (k < from || k >= upto) continue;
            load(delta + t * F, w[k]);
            if constexpr (ONTO)
                if (count <= kPart && rank + 1 == count) load(dW + (long long)row * F, old[k]);
        }
#pragma unroll
        for (int k = 0; k < WINDOW; ++k) {
            const int row = __shfl_sync(0xffffffffu, near.y, k), rank = __shfl_sync(0xffffffffu, near.z, k), count = __shfl_sync(0xffffffffu, near.w, k);
            if (k < from || k >= upto) continue;
            add(w[k]);
            if (rank + 1 != count && rank % kPart != kPart - 1) continue;
            if (count <= kPart) store(row, old[ONTO ? k : 0]);
            else leave(0, k, row, rank, count);
#pragma unroll
            for (int u = 0; u < UN; ++u)
#pragma unroll
                for (int c = 0; c < VEC; ++c) acc[u][c] = 0.0f;
        }
        if (upto > WINDOW) {
            const int row = __shfl_sync(0xffffffffu, near.y, last), rank = __shfl_sync(0xffffffffu, near.z, last) + upto - 1 - last,
                      count = __shfl_sync(0xffffffffu, near.w, last);
            if constexpr (ONTO)
                if (count <= kPart) load(dW + (long long)row * F, old[0]);
            constexpr int AHEAD = UN == 1 ? 8 : 4;
            for (int j = WINDOW; j < upto; j += AHEAD) {
                Pack<T, VEC> x[AHEAD][UN];
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    const int at = j + k;
                    const long long t = __shfl_sync(0xffffffffu, at < 32 ? near.x : far, at & 31);
                    if (at < upto) load(delta + t * F, x[k]);
                }
#pragma unroll
                for (int k = 0; k < AHEAD; ++k)
                    if (j + k < upto) add(x[k]);
            }
            if (count <= kPart) store(row, old[0]);
            else leave(1, upto - 1, row, rank, count);
        }
        if (join_row[0] >= 0 || join_row[1] >= 0) {
            __threadfence();
            __syncwarp();
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                if (join_row[which] < 0) continue;
                const int parts = join_parts[which];
                unsigned came = 0;
                if (lane == 0) came = atomicAdd(a.s.tickets + (long long)join_slot[which] * a.col_blocks + block, 1u);
                if (__shfl_sync(0xffffffffu, came, 0) + 1 != (unsigned)parts) continue;
                __threadfence();
                const float* p = a.s.partial + (long long)join_slot[which] * F + col0;
#pragma unroll
                for (int u = 0; u < UN; ++u) {
                    Sum total[VEC] = {};
                    if (col0 + u * COLS >= F) continue;
                    for (int q = 0; q < parts; q += 8) {
                        float v[8][VEC];
#pragma unroll
                        for (int x = 0; x < 8; ++x)
                            if (q + x < parts) get_sums<VEC>(p + (long long)(q + x) * F + u * COLS, v[x]);
                        if constexpr (flex) {           // (eight parts are at most 2^23)
#pragma unroll
                            for (int c = 0; c < VEC; ++c) {
                                float eight = 0.0f;
#pragma unroll
                                for (int x = 0; x < 8; ++x)
                                    if (q + x < parts) eight += v[x][c];
                                total[c] += (int)eight;
                            }
                        } else {
#pragma unroll
                            for (int x = 0; x < 8; ++x)
                                if (q + x < parts)
#pragma unroll
                                    for (int c = 0; c < VEC; ++c) total[c] += v[x][c];
                        }
                    }
#pragma unroll
                    for (int c = 0; c < VEC; ++c) acc[u][c] = (float)total[c];
                }
                if constexpr (ONTO) load(dW + (long long)join_row[which] * F, old[0]);
                store(join_row[which], old[0]);
            }
        }
    }
    sink.done(f);
}

template <typename T> constexpr int wide() { return 16 / (int)sizeof(T); }

template <typename T, int KIND>
int launch_embed(const void* table, const void* idx, void* out, int V, int F, long long n, float scale, const FlexArgs& f, cudaStream_t st) {
    constexpr int W = wide<T>();
    if (F % W != 0 || !b2::aligned16(table) || !b2::aligned16(out)) {
        constexpr int UN = 8;
        const unsigned col_blocks = (unsigned)((F + 32 * UN - 1) / (32 * UN));
        long long blocks = (n * (long long)col_blocks + 7) / 8;
        if (blocks > (1ll << 30)) blocks = 1ll << 30;
        B2_CUDA((b2::launch_after(embed_apart_kernel<T, KIND, UN>, dim3((unsigned)blocks), 256, 0, st, (const T*)table, idx, (T*)out, V, F, n, col_blocks, scale, f)));
        return B2_OK;
    }
    const long long total = n * (long long)(F / W);
    // four vectors a thread hide the two loads behind one another; where that leaves SMs without a block, one
    const bool deep = total >= 4ll * 256 * b2::kSms;
    long long blocks = (total + (deep ? 1023 : 255)) / (deep ? 1024 : 256);
    if (blocks > (1ll << 30)) blocks = 1ll << 30;
#define B2_EMBED(UN) \
    B2_CUDA((b2::launch_after(embed_kernel<T, W, KIND, UN>, dim3((unsigned)blocks), 256, 0, st, (const T*)table, idx, (T*)out, V, F, n, scale, f)))
    if (deep) B2_EMBED(4);
    else B2_EMBED(1);
#undef B2_EMBED
    return B2_OK;
}

// ---- gradient of few tokens: one launch ---------------------------------------------------------------------------
// A CTA takes its own rows through all steps: its tokens, in order, their numbers within each row, the sums, in parts as
// above, a warp to a row and its columns at a time, and the zeros.  For more tokens the sums want more warps than those of
// the CTA that owns a frequent one.  (256 mantissas add up to 2^23 at most: fp32 holds every sum of them.)
constexpr int kSmall = 256;

__device__ __forceinline__ int token_of_kind(int kind, const void* idx, int i, int V, float step) {
    switch (kind) {
        case B2_IDX_F32: return token_at<B2_IDX_F32>(idx, i, V, step);
        case B2_IDX_I32: return token_at<B2_IDX_I32>(idx, i, V, step);
        case B2_IDX_I64: return token_at<B2_IDX_I64>(idx, i, V, step);
        default: return token_at<B2_IDX_FLEX16>(idx, i, V, step);
    }
}

template <typename T, int VEC, int UN, bool ONTO>
__global__ void __launch_bounds__(512)
small_update_kernel(const T* __restrict__ delta, T* dW, const OrderArgs a, int kind, int F, float scale, const FlexArgs f) {
    extern __shared__ unsigned whole[];         // [rows] tokens of each row
    __shared__ uint2 flat[kSmall];              // position and row of the CTA's tokens
    __shared__ unsigned ranks[kSmall], found_by[kSmall / 32];
    constexpr int COLS = 32 * VEC, WARPS = 512 / 32;
    constexpr bool flex = sizeof(T) == 2;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned G = gridDim.x, b = blockIdx.x;
    const int rows = a.rows;
    for (int i = threadIdx.x; i < rows; i += 512) whole[i] = 0;
    after_earlier_kernels();
    const float istep = kind == B2_IDX_FLEX16 ? a.table[a.slot_idx].scale : 1.0f, step = flex ? f.table[f.slot_in].scale : 1.0f;
    Sink<T, VEC> sink(f);
    int local = 0;
    unsigned those = 0;
    if (warp < kSmall / 32) {
        const int i = threadIdx.x;
        const int v = i < a.n ? token_of_kind(kind, a.idx, i, a.V, istep) : -1;
        local = v / (int)G;
        those = __ballot_sync(0xffffffffu, v >= 0 && v != a.pad && (unsigned)(v - local * (int)G) == b);
        if (lane == 0) found_by[warp] = __popc(those);
    }
    __syncthreads();
    unsigned all = 0, before = 0;
#pragma unroll
    for (int w = 0; w < kSmall / 32; ++w) {
        before += w < warp ? found_by[w] : 0u;
        all += found_by[w];
    }
    if (those >> lane & 1u) flat[before + __popc(those & ((1u << lane) - 1u))] = make_uint2(threadIdx.x, (unsigned)local);
    __syncthreads();
    if (warp == 0)
        for (unsigned k = lane; k - lane < all; k += 32) {
            const unsigned mine = k < all ? flat[k].y : 0xffffffffu;
            const unsigned same = __match_any_sync(0xffffffffu, mine);
            const unsigned c = k < all ? whole[mine] : 0u, place = __popc(same & ((1u << lane) - 1u));
            __syncwarp();
            if (k < all) {
                ranks[k] = c + place;
                if (place == 0) whole[mine] = c + __popc(same);
            }
            __syncwarp();
        }
    __syncthreads();
    for (unsigned unit = warp; unit < all * (unsigned)a.col_blocks; unit += WARPS) {
        const unsigned first = unit / (unsigned)a.col_blocks;
        if (ranks[first] != 0) continue;        // (a row is taken up where its first token stands)
        const unsigned mine = flat[first].y;
        const int count = (int)whole[mine], col0 = (int)(unit - first * a.col_blocks) * COLS * UN + lane * VEC;
        T* to = dW + ((long long)b + (long long)mine * G) * F + col0;
        Pack<T, VEC> old[UN];
        if constexpr (ONTO)
#pragma unroll
            for (int u = 0; u < UN; ++u)
                if (col0 + u * COLS < F) old[u].load(to + u * COLS);
        float acc[UN][VEC] = {}, sum[UN][VEC] = {};
        int done = 0;
        for (unsigned j0 = first; done < count; j0 += 32) {
            const uint2 e = j0 + lane < all ? flat[j0 + lane] : make_uint2(0, 0xffffffffu);
            unsigned left = __ballot_sync(0xffffffffu, e.y == mine);
            while (left) {
                constexpr int AHEAD = UN == 1 ? 8 : 4;
                Pack<T, VEC> w[AHEAD][UN];
                const int now = min(AHEAD, __popc(left));
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    const long long t = __shfl_sync(0xffffffffu, e.x, left ? __ffs(left) - 1 : 0);
                    left &= left - 1;
                    if (k < now)
#pragma unroll
                        for (int u = 0; u < UN; ++u)
                            if (col0 + u * COLS < F) w[k][u].load(delta + t * F + col0 + u * COLS);
                }
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    if (k >= now) break;
#pragma unroll
                    for (int u = 0; u < UN; ++u)
                        if (col0 + u * COLS < F) {
                            float v[VEC];
                            w[k][u].get(v);
#pragma unroll
                            for (int c = 0; c < VEC; ++c) acc[u][c] += v[c];
                        }
                    if (++done % kPart == 0 || done == count)
#pragma unroll
                        for (int u = 0; u < UN; ++u)
#pragma unroll
                            for (int c = 0; c < VEC; ++c) {
                                sum[u][c] = done <= kPart ? acc[u][c] : sum[u][c] + acc[u][c];
                                acc[u][c] = 0.0f;
                            }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            if (col0 + u * COLS >= F) continue;
            float v[VEC];
#pragma unroll
            for (int c = 0; c < VEC; ++c) v[c] = flex ? (sum[u][c] * step) * scale : sum[u][c] * scale;
            if constexpr (ONTO) {
                float o[VEC];
                old[u].get(o);
#pragma unroll
                for (int c = 0; c < VEC; ++c) v[c] = o[c] + v[c];
            }
            sink.put(to + u * COLS, v);
        }
    }
    if (!ONTO && !f.probe)
        for (int r = warp; r < rows; r += WARPS) {
            const long long row = (long long)b + (long long)r * G;
            if (row < a.V && whole[r] == 0) zero_row(dW + row * F, F, lane);
        }
    sink.done(f);
}

// Columns of a warp: 16 bytes to a lane, or four values apart where rows are not aligned.
constexpr int kApart = 4;
int col_blocks_of(int F, int vec) {
    const int cols = vec > 1 ? 32 * vec : 32 * kApart;
    return (F + cols - 1) / cols;
}

template <int KIND>
int launch_order(const OrderArgs& a, int owners, cudaStream_t st) {
    static std::atomic<unsigned long long> done{0};
    B2_CHECK(b2::allow_shared((const void*)order_kernel<KIND>, kCounters * 4, &done));
    const size_t many = (size_t)a.rows * (a.stride + 2) * 4, few = (size_t)(2 * a.rows + 3) / 4 * 16 + kOrderThreads / 32 * kListed * 8 + kFlat * 12;
    B2_CUDA((b2::launch_after(order_kernel<KIND>, dim3((unsigned)owners), kOrderThreads, many > few ? many : few, st, a)));
    return B2_OK;
}

template <typename T>
int launch_update(const void* delta, const void* idx, void* dW, int kind, int V, int F, long long n, float scale, int pad, int onto, const FlexArgs& f,
                  void* scratch, cudaStream_t st) {
    if (n == 0 && (onto || f.probe)) return B2_OK;
    // (four values to a lane of either type: with eight mantissas 16384 x 1024 into 30000 rows took 52 us, 49 so; 16384 x 64
    // into 200 rows 26 and 21)
    constexpr int W = 4;
    const bool vec = F % W == 0 && ((uintptr_t)delta | (uintptr_t)dW) % (W * sizeof(T)) == 0;
    const int owners = owners_of(V);
    OrderArgs a;
    a.idx = idx;
    a.V = V;
    a.n = (int)n;
    a.pad = pad;
    a.rows = (V + owners - 1) / owners;
    a.warps = kCounters / a.rows - 3;           // (a word for each, made odd, and two more)
    if (a.warps > kOrderThreads / 32) a.warps = kOrderThreads / 32;
    a.stride = a.warps | 1;
    a.magic = owners == 1 ? 0u : (unsigned)((1ull << 32) / owners + 1);     // (one owner has one row)
    a.col_blocks = col_blocks_of(F, vec ? W : 1);
    a.s = scratch_of(scratch, V, F, n, a.col_blocks);
    a.table = f.table;
    a.slot_idx = f.slot_idx;
    if (n <= kSmall) {
#define B2_SMALL(VEC, UN, ONTO)                                                                                                              \
    B2_CUDA((b2::launch_after(small_update_kernel<T, VEC, UN, ONTO>, dim3((unsigned)owners), 512, (size_t)a.rows * 4, st, (const T*)delta, (T*)dW, a, kind, \
                              F, scale, f)))
        if constexpr (sizeof(T) == 4) {
            if (onto && vec) B2_SMALL(W, 1, true);
            else if (onto) B2_SMALL(1, kApart, true);
        }
        if (!onto && vec) B2_SMALL(W, 1, false);
        else if (!onto) B2_SMALL(1, kApart, false);
#undef B2_SMALL
        return B2_OK;
    }
    switch (kind) {
        case B2_IDX_F32: B2_CHECK(launch_order<B2_IDX_F32>(a, owners, st)); break;
        case B2_IDX_I32: B2_CHECK(launch_order<B2_IDX_I32>(a, owners, st)); break;
        case B2_IDX_I64: B2_CHECK(launch_order<B2_IDX_I64>(a, owners, st)); break;
        default: B2_CHECK(launch_order<B2_IDX_FLEX16>(a, owners, st));
    }
    // Windows of 8 places where these occupy the machine and nothing else is loaded, of 4 elsewhere (8192 x 1024 into
    // 32000 rows 32.6 us a call, 34.0 with 4; onto them 20.3 and 19.2; 3001 x 301 flex16 17.1 and 15.5; 2000 x 1024 into
    // 200 rows 12.6 and 11.5).  Of 2: 38, 22, 15.0 and 11.5.
    auto blocks_of = [&](int window) { return (n + kSumWarps * window - 1) / (kSumWarps * window) * a.col_blocks; };
    const bool longer = vec && !onto && blocks_of(8) >= 8 * b2::kSms;
    const long long sum_blocks = blocks_of(longer ? 8 : 4);
    // about 4 KB of zeros to a warp (16: 3001 x 301 flex16 into 10007 rows 22 us, 15 with 4)
    const long long fit = 4096 / ((long long)F * (long long)sizeof(T));
    const int zero_rows = fit < 1 ? 1 : fit > 32 ? 32 : (int)fit;
    const long long zero_blocks = onto || f.probe ? 0 : ((long long)owners * a.rows + kSumWarps * zero_rows - 1) / (kSumWarps * zero_rows);
    B2_REQUIRE(sum_blocks + zero_blocks < (1ll << 31), "%lld tokens of %d features are too many for one launch", n, F);
    const SumArgs sa = {V, F, (int)n, a.rows, owners, zero_rows, (unsigned)a.col_blocks, (unsigned)sum_blocks, scale, a.s};
    const dim3 grid((unsigned)(sum_blocks + zero_blocks));
#define B2_SUM(VEC, UN, WINDOW, ONTO) \
    B2_CUDA((b2::launch_after(sum_kernel<T, VEC, UN, WINDOW, ONTO>, grid, 32 * kSumWarps, 0, st, (const T*)delta, (T*)dW, sa, f)))
    if constexpr (sizeof(T) == 4) {
        if (onto && vec) B2_SUM(W, 1, 4, true);
        else if (onto) B2_SUM(1, kApart, 4, true);
    }
    if (longer) B2_SUM(W, 1, 8, false);
    else if (!onto && vec) B2_SUM(W, 1, 4, false);
    else if (!onto) B2_SUM(1, kApart, 4, false);
#undef B2_SUM
    return B2_OK;
}

int check_flex(int flex, int kind, const FlexArgs& f) {
    B2_REQUIRE(kind >= B2_IDX_F32 && kind <= B2_IDX_FLEX16, "unknown kind of index: %d", kind);
    B2_REQUIRE(kind != B2_IDX_FLEX16 || (f.table && f.slot_idx >= 0), "a flex16 index needs the scale table");
    B2_REQUIRE((!flex && kind != B2_IDX_FLEX16) || (uintptr_t)f.table % alignof(b2_flex_scale) == 0, "the scale table lies between two addresses");
    if (!flex) return B2_OK;
    B2_REQUIRE(f.table && f.slot_in >= 0 && f.slot_out >= 0, "a flex16 lookup needs the scale table");
    B2_REQUIRE(f.probe ? f.probe_out != nullptr : f.stats != nullptr, "missing statistics destination");
    B2_REQUIRE((f.probe ? (uintptr_t)f.probe_out % 8 : (uintptr_t)f.stats % 4) == 0, "the statistics lie between two addresses");
    return B2_OK;
}

// Exponents that the kernels read, and the words that they keep the largest value in.
int check_flex_memory(b2::Memory& memory, int flex, int kind, const FlexArgs& f) {
    if (flex || kind == B2_IDX_FLEX16) B2_CHECK(memory.read(f.table, "the scale table"));
    if (!flex) return B2_OK;
    if (f.probe) return memory.written(f.probe_out, "the word of a measuring launch");
    return memory.written(f.stats, "the statistics");
}

}  // namespace

static int check_memory(const void* whole, int32_t V, const void* rows, int64_t n, int32_t F, const void* idx, int32_t idx_kind, int32_t flex,
                        bool whole_written) {
    const size_t value = flex ? 2 : 4, token = idx_kind == B2_IDX_I64 ? 8 : idx_kind == B2_IDX_FLEX16 ? 2 : 4;
    B2_REQUIRE((uintptr_t)whole % value == 0 && (uintptr_t)rows % value == 0 && (uintptr_t)idx % token == 0, "a tensor of the lookup lies between two addresses");
    const size_t table = (size_t)V * F * value, list = (size_t)n * F * value, tokens = (size_t)n * token;
    B2_REQUIRE(!b2::overlap(whole, table, rows, list) &&
                   !(whole_written ? b2::overlap(whole, table, idx, tokens) : b2::overlap(rows, list, idx, tokens)),
               "the result of the lookup, or of its gradient, overlaps an operand");
    return B2_OK;
}

extern "C" int b2_embed_fprop(const void* table, const void* idx, void* out, int32_t flex, int32_t idx_kind, int32_t V, int32_t F, int64_t n_idx,
                              float scale, const b2_flex_scale* scales, int32_t slot_table, int32_t slot_idx, int32_t slot_out, int32_t* stats,
                              uint64_t* probe_out, int32_t probe, void* stream) {
    B2_REQUIRE(V > 0 && F > 0 && n_idx >= 0, "bad lookup: table %d x %d, %lld tokens", V, F, (long long)n_idx);
    const FlexArgs f = {scales, slot_table, slot_idx, slot_out, stats, (unsigned long long*)probe_out, probe ? 1 : 0};
    B2_CHECK(check_flex(flex, idx_kind, f));
    if (n_idx == 0) return B2_OK;
    B2_REQUIRE(table && idx && out, "bad lookup: missing tensor");
    B2_CHECK(check_memory(table, V, out, n_idx, F, idx, idx_kind, flex, false));
    b2::Memory memory;
    B2_CHECK(memory.find_device());
    B2_CHECK(memory.written(out, "the lookup's result"));
    B2_CHECK(memory.read(table, "the table"));
    B2_CHECK(memory.read(idx, "the index"));
    B2_CHECK(check_flex_memory(memory, flex, idx_kind, f));
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
    *bytes = scratch_of(nullptr, V, F, n_idx, col_blocks_of(F, 1)).bytes + 256;
    return B2_OK;
}

extern "C" int b2_embed_update_launches(int64_t n_idx, int32_t* launches) {
    B2_REQUIRE(launches && n_idx >= 0, "bad argument");
    *launches = n_idx <= kSmall ? 1 : 2;
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
    B2_CHECK(check_memory(dW, V, delta, n_idx, F, idx, idx_kind, flex, true));
    const size_t value = flex ? 2 : 4, token = idx_kind == B2_IDX_I64 ? 8 : idx_kind == B2_IDX_FLEX16 ? 2 : 4;
    B2_REQUIRE(!b2::overlap(scratch, need, dW, (size_t)V * F * value) && !b2::overlap(scratch, need, delta, (size_t)n_idx * F * value) &&
                   !b2::overlap(scratch, need, idx, (size_t)n_idx * token),
               "the scratch overlaps a tensor of the lookup's gradient");
    b2::Memory memory;
    B2_CHECK(memory.find_device());
    B2_CHECK(memory.written(dW, "the table's gradient"));
    B2_CHECK(memory.written(scratch, "the scratch"));
    B2_CHECK(memory.read(n_idx ? delta : nullptr, "delta"));
    B2_CHECK(memory.read(n_idx ? idx : nullptr, "the index"));
    B2_CHECK(check_flex_memory(memory, flex, idx_kind, f));
    const int pad = pad_idx >= 0 && pad_idx < V ? (int)pad_idx : -1;
    void* at = (void*)(((uintptr_t)scratch + 255) / 256 * 256);
    if (flex) return launch_update<short>(delta, idx, dW, idx_kind, V, F, n_idx, scale, pad, onto, f, at, (cudaStream_t)stream);
    return launch_update<float>(delta, idx, dW, idx_kind, V, F, n_idx, scale, pad, onto ? 1 : 0, f, at, (cudaStream_t)stream);
}
