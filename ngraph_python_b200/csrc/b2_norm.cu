// The edge between two blocks of a residual network, and its gradients:
//
//   stream = a residual + gate * (rms(block) * w_post),   out = rms(stream) * w_pre,   rms(x) = x * rstd(x)
//
//   d_stream' = d_stream + through(d_out, stream, w_pre),  d_residual = a d_stream',  d_gate = d_stream' * rms(block) w_post
//   d_block   = through(gate * d_stream', block, w_post)
//   through(d, x, w) = rstd (w d - x^ mean(w d x^)),  x^ = x rstd;   d_w = sum over rows of d x^
//
// Bound by memory: four tensors of rows forward, six for the gradients, each read or written once.  8192 x 4096: 86 us
// forward, 0.96 of the rate of a copy, 134 us for the gradients, 0.92.  One row of 2048: 2.3 us in a graph.
#include <cstdint>
#include <utility>

#include "b2_operators.h"
#include "b2_ew_device.cuh"

namespace {

using b2::Rows;
using b2::rows_at;
using b2::check_apart;

constexpr int kThreads = 512;        // of a CTA for rows of any length

// VEC values next to one another
template <int VEC>
__device__ __forceinline__ void get(const float* p, float* v) {
    if constexpr (VEC == 4) {
        const float4 w = *reinterpret_cast<const float4*>(p);
        v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
    } else {
        v[0] = *p;
    }
}
template <int VEC>
__device__ __forceinline__ void put(float* p, const float* v) {
    if constexpr (VEC == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else *p = v[0];
}

// values that a pointer is behind a 16-byte boundary
__device__ __host__ __forceinline__ int shift_of(const float* p) { return (int)((reinterpret_cast<uintptr_t>(p) >> 2) & 3); }

// Sums of up to two values over the CTA, the same bits in every thread.  One barrier: calls write to two sets of words by
// turns, and who comes to write to a set again has passed the barrier behind which everybody had read it.
struct TwoSums {
    float words[2][2][32];
};
template <int N>
__device__ __forceinline__ void cta_sums(float (&x)[N], TwoSums& s, int& turn) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < N; ++k) x[k] += __shfl_xor_sync(0xffffffffu, x[k], o);
    if (lane == 0)
#pragma unroll
        for (int k = 0; k < N; ++k) s.words[turn][k][warp] = x[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = lane < warps ? s.words[turn][k][lane] : 0.0f;
    for (int o = warps > 16 ? 16 : warps > 8 ? 8 : warps > 4 ? 4 : warps > 2 ? 2 : warps - 1; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < N; ++k) x[k] += __shfl_xor_sync(0xffffffffu, x[k], o);
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = __shfl_sync(0xffffffffu, x[k], 0);
    turn ^= 1;
}

__device__ __forceinline__ float block_sum(float v, float* words) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) words[warp] = v;
    __syncthreads();
    v = 0.0f;
    for (int w = 0; w < (int)(blockDim.x >> 5); ++w) v += words[w];
    return v;
}

__device__ __forceinline__ float rstd_of(float squares, int F, float eps) { return __frsqrt_rn(__fdividef(squares, (float)F) + eps); }

__device__ __forceinline__ float gate_at(const b2_norm& a, long long row, int i) {
    switch (a.gate_kind) {
        case B2_GATE_FEATURE: return a.gate[i];
        case B2_GATE_ROW: return a.gate[row];
        case B2_GATE_FULL: return a.gate[row * a.gate_stride + i];
        default: return 1.0f;
    }
}

// Rows of any length and alignment: what a row's sums need is read again.
template <int VEC>
__global__ void __launch_bounds__(kThreads)
norm_any_kernel(const b2_norm a) {
    __shared__ float words[32];
    after_earlier_kernels();
    const int F = a.features;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float* u = a.block ? a.block + row * a.block_stride : nullptr;
        const float* r = a.residual + row * a.residual_stride;
        float* s = a.block ? a.stream + row * a.stream_stride : nullptr;
        float rho = 1.0f;
        if (a.post_weight) {
            float q = 0.0f;
            for (int i = threadIdx.x * VEC; i < F; i += kThreads * VEC) {
                float y[VEC];
                get<VEC>(u + i, y);
#pragma unroll
                for (int j = 0; j < VEC; ++j) q = fmaf(y[j], y[j], q);
            }
            rho = rstd_of(block_sum(q, words), F, a.eps);
            if (a.block_rstd && threadIdx.x == 0) a.block_rstd[row] = rho;
        }
        float q = 0.0f;
        for (int i = threadIdx.x * VEC; i < F; i += kThreads * VEC) {
            float x[VEC], y[VEC];
            get<VEC>(r + i, x);
            if (u) {
                get<VEC>(u + i, y);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    if (a.post_weight) y[j] = y[j] * rho * a.post_weight[i + j];
                    x[j] = fmaf(y[j], gate_at(a, row, i + j), a.residual_scale * x[j]);
                }
                put<VEC>(s + i, x);
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) q = fmaf(x[j], x[j], q);
        }
        if (!a.out && !a.stream_rstd) continue;
        rho = rstd_of(block_sum(q, words), F, a.eps);
        if (a.stream_rstd && threadIdx.x == 0) a.stream_rstd[row] = rho;
        if (a.out)
            for (int i = threadIdx.x * VEC; i < F; i += kThreads * VEC) {
                float x[VEC];
                get<VEC>((s ? s : r) + i, x);
#pragma unroll
                for (int j = 0; j < VEC; ++j) x[j] = x[j] * rho * a.pre_weight[i + j];
                put<VEC>(a.out + row * a.out_stride + i, x);
            }
    }
}

// The first of a thread's IT vectors of a row: they are 32 vectors apart, a distance that addresses take as a constant.
template <int VEC, int IT>
__device__ __forceinline__ int first_of() { return ((int)(threadIdx.x >> 5) * IT * 32 + (int)(threadIdx.x & 31)) * VEC; }

// A thread's vectors of a row.  Where rows are not aligned but all tensors' rows lie alike, some values behind a 16-byte
// boundary, the vectors are those of memory, and the row's two ends are taken value by value -- behind all vectors,
// since a branch between two loads keeps the second waiting.
template <int VEC, int IT, bool RAGGED>
__device__ __forceinline__ void get_row(const float* row, int i0, int F, float (*v)[VEC]) {
#pragma unroll
    for (int k = 0; k < IT; ++k) {
        const int i = i0 + k * 32 * VEC;
        if (RAGGED ? i >= 0 && i + VEC <= F : i < F) get<VEC>(row + i, v[k]);
    }
    if constexpr (RAGGED)
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const int i = i0 + k * 32 * VEC;
            if (i < 0 || (i < F && i + VEC > F))
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[k][j] = i + j >= 0 && i + j < F ? row[i + j] : 0.0f;
        }
}
template <int VEC, int IT, bool RAGGED>
__device__ __forceinline__ void put_row(float* row, int i0, int F, const float (*v)[VEC]) {
#pragma unroll
    for (int k = 0; k < IT; ++k) {
        const int i = i0 + k * 32 * VEC;
        if (RAGGED ? i >= 0 && i + VEC <= F : i < F) put<VEC>(row + i, v[k]);
    }
    if constexpr (RAGGED)
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const int i = i0 + k * 32 * VEC;
            if (i < 0 || (i < F && i + VEC > F))
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (i + j >= 0 && i + j < F) row[i + j] = v[k][j];
        }
}

__device__ __forceinline__ void fetch_ahead(const float* p, int bytes) {
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

// A row to a CTA, held in registers: each tensor is read once.  Both operands are on their way before the first sum.
// Ragged rows: a CTA's are a multiple of four apart and so lie alike, and it keeps the weights in shared memory as they
// lie beside them.
template <int IT, bool RAGGED, bool U, bool POST, int GATE>
__global__ void __launch_bounds__(1024)
norm_row_kernel(const b2_norm a) {
    extern __shared__ __align__(16) float staged[];         // ragged: post_weight, a gate per feature, pre_weight
    __shared__ TwoSums sums;
    after_earlier_kernels();
    constexpr int VEC = 4, di = 32 * VEC;
    const int F = a.features, width = (F + 6) / 4 * 4;
    const int shift = RAGGED ? shift_of(a.residual + blockIdx.x * a.residual_stride) : 0, i0 = first_of<VEC, IT>() - shift;
    if (RAGGED) {
        for (int i = threadIdx.x; i < width; i += blockDim.x) {
            const bool there = i >= shift && i - shift < F;
            if (POST) staged[i] = there ? a.post_weight[i - shift] : 0.0f;
            if (GATE == B2_GATE_FEATURE) staged[width + i] = there ? a.gate[i - shift] : 0.0f;
            if (a.out) staged[2 * width + i] = there ? a.pre_weight[i - shift] : 0.0f;
        }
        __syncthreads();
    }
    auto get_weights = [&](int which, const float* w, int i, float* v) {
        if (RAGGED ? i + shift < width : i < F) get<VEC>(RAGGED ? staged + which * width + i + shift : w + i, v);
    };
    int turn = 0;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float x[IT][VEC] = {}, u[IT][VEC] = {};
        const float* r = a.residual + row * a.residual_stride;
        if (U) get_row<VEC, IT, RAGGED>(a.block + row * a.block_stride, i0, F, u);
        get_row<VEC, IT, RAGGED>(r, i0, F, x);
        if (RAGGED && threadIdx.x == 0 && row + gridDim.x < a.rows) {
            // the next row on its way to the second cache
            const long long next = row + gridDim.x;
            const int bytes = (shift + F + 3) / 4 * 16;         // (whole vectors, the last with the row's last value)
            fetch_ahead(a.residual + next * a.residual_stride - shift, bytes);
            if (U) fetch_ahead(a.block + next * a.block_stride - shift, bytes);
        }
        if constexpr (U) {
            float rho = 1.0f;
            if (POST) {
                float q[1] = {0.0f};
#pragma unroll
                for (int k = 0; k < IT; ++k)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) q[0] = fmaf(u[k][j], u[k][j], q[0]);
                cta_sums(q, sums, turn);
                rho = rstd_of(q[0], F, a.eps);
                if (a.block_rstd && threadIdx.x == 0) a.block_rstd[row] = rho;
            }
            if (GATE == B2_GATE_ROW) rho *= a.gate[row];
#pragma unroll
            for (int k = 0; k < IT; ++k) {
                const int i = i0 + k * di;
                float w[VEC], g[1][VEC];
                if (POST) get_weights(0, a.post_weight, i, w);
                if (GATE == B2_GATE_FULL) get_row<VEC, 1, RAGGED>(a.gate + row * a.gate_stride, i, F, g);
                if (GATE == B2_GATE_FEATURE) get_weights(1, a.gate, i, g[0]);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    float y = POST || GATE == B2_GATE_ROW ? u[k][j] * rho : u[k][j];
                    if (POST) y *= w[j];
                    if (GATE == B2_GATE_FULL || GATE == B2_GATE_FEATURE) y *= g[0][j];
                    x[k][j] = fmaf(a.residual_scale, x[k][j], y);
                    if (i + j >= F || (RAGGED && i + j < 0)) x[k][j] = 0.0f;
                }
            }
            put_row<VEC, IT, RAGGED>(a.stream + row * a.stream_stride, i0, F, x);
        }
        if (!a.out && !a.stream_rstd) continue;
        float q[1] = {0.0f};
#pragma unroll
        for (int k = 0; k < IT; ++k)
#pragma unroll
            for (int j = 0; j < VEC; ++j) q[0] = fmaf(x[k][j], x[k][j], q[0]);
        cta_sums(q, sums, turn);
        const float rho = rstd_of(q[0], F, a.eps);
        if (a.stream_rstd && threadIdx.x == 0) a.stream_rstd[row] = rho;
        if (!a.out) continue;
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const int i = i0 + k * di;
            float w[VEC];
            get_weights(2, a.pre_weight, i, w);
#pragma unroll
            for (int j = 0; j < VEC; ++j) x[k][j] = x[k][j] * rho * w[j];
        }
        put_row<VEC, IT, RAGGED>(a.out + row * a.out_stride, i0, F, x);
    }
}

// Gradients, a row to a CTA at a time.  A CTA keeps its rows' sums for the weights and a gate per feature in registers.
// The tensors of its next rows are on their way into shared memory meanwhile (bulk copies; a ring of `stages` rows),
// since between the loads of a row and its stores there are two sums over the CTA: the first pair (stream, d_out) of a
// place is free again behind the first of them, the others behind the second.  Ragged rows: a CTA's are a multiple of four
// apart and so lie alike; a copy starts at the 16-byte boundary below the row, and a thread's columns, whose sums it keeps,
// are the vectors of memory.  (Value by value 3000 x 5001 took 83 us.)
constexpr int kStages = 3;
constexpr int kGradShared = 226 << 10;      // (of 227 KB, with the static words)

struct Ring {
    int stages, slot;                   // bytes of one tensor's row, with room for its alignment
};

// Waits are bounded.  When one has run out, no thread of the CTA waits any more and thread 0 asks for no more rows; at the end
// the CTA's results are spoiled.
struct Waits {
    unsigned long long first_full[kStages], then_full[kStages];
    int ran_out;                        // 1: a wait has run out; 2, 3: of thread 0, for the first or the other tensors of row `stopped`
    long long stopped;
};

// Sets *status and turns all results of the CTA's rows, and its sums, into NaN.  Copies that are still on their way are waited
// for once more: the shared memory is another CTA's then.  (A call, which leaves the registers of the rows' loop alone: inlined,
// 16384 x 2047 with a gate for a row took 180 us, 152 so.)
__device__ __noinline__ void spoil_rows(const b2_norm& a, const b2_norm_grads& d, float* mine, Waits& waits, int stages, bool two) {
    if (threadIdx.x == 0) {
        // thread 0 asks for the tensors of the row `stages` ahead behind each of its two waits
        const int rows = (int)((a.rows - 1 - blockIdx.x) / gridDim.x) + 1, at = (int)((waits.stopped - blockIdx.x) / gridDim.x) + stages;
        for (int which = 0; waits.ran_out >= 2 && which < (two ? 2 : 1); ++which) {
            const int asked = min(rows, at + (which == 0 && waits.ran_out == 3));
            for (int n = max(0, asked - stages); n < asked; ++n) b2_mbar_wait((which ? waits.then_full : waits.first_full) + n % stages, n / stages & 1);
        }
        if (d.status) atomicExch(d.status, 1);
    }
    const float nan = __int_as_float(0x7fffffff);
    const bool full = a.gate_kind == B2_GATE_FULL;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        for (int i = threadIdx.x; i < a.features; i += blockDim.x) {
            if (d.d_residual) d.d_residual[row * d.d_residual_stride + i] = nan;
            if (d.d_block) d.d_block[row * d.d_block_stride + i] = nan;
            if (full && d.d_gate) d.d_gate[row * d.d_gate_stride + i] = nan;
        }
        if (a.gate_kind == B2_GATE_ROW && d.d_gate && threadIdx.x == 0) d.d_gate[row] = nan;
    }
    for (int i = threadIdx.x; i < 3 * a.features; i += blockDim.x) mine[i] = nan;
    __syncthreads();
}

// (One CTA as the least: left to itself the assembler gives some of these so few registers that they spill.)
template <bool RAGGED, int MOST, int IT, bool U, bool POST, int GATE>
__global__ void __launch_bounds__(MOST, 1)
norm_grad_row_kernel(const __grid_constant__ b2_norm a, const __grid_constant__ b2_norm_grads d, float* __restrict__ out_sums, const Ring ring) {
    extern __shared__ __align__(128) unsigned char shared[];
    __shared__ Waits waits;
    __shared__ TwoSums sums;
    constexpr int VEC = 4;
    constexpr bool HOLD = IT == 2;              // weights stay in registers, in shared memory otherwise
    constexpr bool FULL = GATE == B2_GATE_FULL, FEATURE = GATE == B2_GATE_FEATURE;
    const bool has_ds = d.d_stream != nullptr;
    // places of the tensors within a stage
    const int at_dy = ring.slot, at_ds = 2 * ring.slot, at_u = at_ds + (has_ds ? ring.slot : 0), at_g = at_u + (U ? ring.slot : 0);
    const int stage_bytes = at_g + (FULL ? ring.slot : 0);
    unsigned char* const room = shared + (HOLD ? 0 : (1 + POST + FEATURE) * ring.slot);
    const float* xs = U ? a.stream : a.residual;
    const long long xs_stride = U ? a.stream_stride : a.residual_stride;
    const int F = a.features, tid = threadIdx.x, shift = RAGGED ? shift_of(xs + blockIdx.x * xs_stride) : 0, i0 = first_of<VEC, IT>() - shift;
    if (tid == 0) {
        for (int s = 0; s < ring.stages; ++s) {
            b2_mbar_init(waits.first_full + s, 1);
            b2_mbar_init(waits.then_full + s, 1);
        }
        b2_mbar_init_fence();
        waits.ran_out = 0;
    }
    __syncthreads();
    after_earlier_kernels();

    auto bytes_of = [&](const float* p) { return (unsigned)((shift_of(p) + F + 3) / 4 * 16); };
    auto copy = [&](const float* p, int to, unsigned long long* bar) { b2_bulk_g2s(room + to, p - shift_of(p), bytes_of(p), bar); };
    auto fetch_first = [&](long long row, int s) {
        const float *x = xs + row * xs_stride, *dy = d.d_out + row * d.d_out_stride;
        b2_mbar_expect_tx(waits.first_full + s, bytes_of(x) + bytes_of(dy));
        copy(x, s * stage_bytes, waits.first_full + s);
        copy(dy, s * stage_bytes + at_dy, waits.first_full + s);
    };
    auto fetch_then = [&](long long row, int s) {
        const float *ds = has_ds ? d.d_stream + row * d.d_stream_stride : nullptr, *u = U ? a.block + row * a.block_stride : nullptr,
                    *g = FULL ? a.gate + row * a.gate_stride : nullptr;
        if (!ds && !u && !g) return;
        b2_mbar_expect_tx(waits.then_full + s, (ds ? bytes_of(ds) : 0u) + (u ? bytes_of(u) : 0u) + (g ? bytes_of(g) : 0u));
        if (ds) copy(ds, s * stage_bytes + at_ds, waits.then_full + s);
        if (u) copy(u, s * stage_bytes + at_u, waits.then_full + s);
        if (g) copy(g, s * stage_bytes + at_g, waits.then_full + s);
    };
    if (tid == 0)
        for (int s = 0; s < ring.stages; ++s) {
            const long long row = blockIdx.x + (long long)s * gridDim.x;
            if (row < a.rows) {
                fetch_first(row, s);
                fetch_then(row, s);
            }
        }

    float sum_pre[IT][VEC] = {}, sum_post[IT][VEC] = {}, sum_gate[IT][VEC] = {};
    float w_pre[IT][VEC] = {}, w_post[IT][VEC] = {}, w_gate[IT][VEC] = {};
    // vectors that reach beyond the row's ends: values of no row are zero, and are not stored
    auto cut = [&](int i) { return RAGGED && (i < 0 || i + VEC > F); };
    auto load = [&](const float* p, int i, float* v) {
        get<VEC>(p + i, v);
        if (cut(i))
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (i + j < 0 || i + j >= F) v[j] = 0.0f;
    };
    auto store = [&](float* p, int i, const float* v) {
        if (!cut(i)) {
            put<VEC>(p + i, v);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (i + j >= 0 && i + j < F) p[i + j] = v[j];
        }
    };
    auto weight = [&](const float* w, int i, float* v) {
        if (RAGGED) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = i + j >= 0 && i + j < F ? w[i + j] : 0.0f;
        } else if (i < F) {
            get<VEC>(w + i, v);
        }
    };
    // (each thread keeps and reads its own columns)
    float* const kept = reinterpret_cast<float*>(shared) + shift;
    const int apart = ring.slot / (int)sizeof(float);
#pragma unroll
    for (int k = 0; k < IT; ++k) {
        const int i = i0 + k * 32 * VEC;
        weight(a.pre_weight, i, w_pre[k]);
        if (POST) weight(a.post_weight, i, w_post[k]);
        if (FEATURE) weight(a.gate, i, w_gate[k]);
        if (!HOLD && i < F) {
            put<VEC>(kept + i, w_pre[k]);
            if (POST) put<VEC>(kept + apart + i, w_post[k]);
            if (FEATURE) put<VEC>(kept + (POST ? 2 : 1) * apart + i, w_gate[k]);
        }
    }
    const float over = 1.0f / (float)F;
    int turn = 0, s = 0;
    unsigned phase = 0;
    auto wait = [&](unsigned long long* bar, long long row, bool first) {
        if (b2_mbar_try_wait(bar, phase)) return;
        for (int i = 0; i < (1 << 22) && *(volatile int*)&waits.ran_out == 0; ++i)
            if (b2_mbar_try_wait(bar, phase)) return;
        if (tid == 0 && waits.ran_out < 2) waits.stopped = row;
        if (tid != 0 || waits.ran_out < 2) atomicMax(&waits.ran_out, tid != 0 ? 1 : first ? 2 : 3);
    };
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const long long next = row + (long long)ring.stages * gridDim.x;
        const unsigned char* here = room + s * stage_bytes;
        float t[IT][VEC] = {};
        const float rho = a.stream_rstd[row], rho_u = POST ? a.block_rstd[row] : 1.0f;
        const float row_gate = GATE == B2_GATE_ROW ? a.gate[row] : 1.0f;
        {
            wait(waits.first_full + s, row, true);
            const float *x = reinterpret_cast<const float*>(here) + shift, *dy = reinterpret_cast<const float*>(here + at_dy) + shift;
            float xh[IT][VEC];
            float q[1] = {0.0f};
#pragma unroll
            for (int k = 0; k < IT; ++k) {
                const int i = i0 + k * 32 * VEC;
                float v[VEC] = {}, y[VEC] = {};
                if (i < F) {
                    if constexpr (!HOLD) get<VEC>(kept + i, w_pre[k]);
                    load(x, i, v);
                    load(dy, i, y);
                }
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    xh[k][j] = v[j] * rho;
                    sum_pre[k][j] = fmaf(y[j], xh[k][j], sum_pre[k][j]);
                    t[k][j] = y[j] * w_pre[k][j];
                    q[0] = fmaf(t[k][j], xh[k][j], q[0]);
                }
            }
            cta_sums(q, sums, turn);
            if (tid == 0 && next < a.rows && waits.ran_out < 2) fetch_first(next, s);
            const float mean = q[0] * over;
#pragma unroll
            for (int k = 0; k < IT; ++k)
#pragma unroll
                for (int j = 0; j < VEC; ++j) t[k][j] = rho * fmaf(xh[k][j], -mean, t[k][j]);
        }
        if (has_ds || U) wait(waits.then_full + s, row, false);
        const float *ds = reinterpret_cast<const float*>(here + at_ds) + shift, *u = reinterpret_cast<const float*>(here + at_u) + shift,
                    *g = reinterpret_cast<const float*>(here + at_g) + shift;
        float uh[IT][VEC] = {};
        float dots[2] = {0.0f, 0.0f};               // of the block's norm, of a row's gate
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const int i = i0 + k * 32 * VEC;
            if (i >= F) continue;
            float v[VEC];
            if (has_ds) {
                load(ds, i, v);
#pragma unroll
                for (int j = 0; j < VEC; ++j) t[k][j] += v[j];
            }
            if (d.d_residual) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = a.residual_scale * t[k][j];
                store(d.d_residual + row * d.d_residual_stride, i, v);
            }
            if constexpr (!U) continue;
            if constexpr (!HOLD) {
                if (POST) get<VEC>(kept + apart + i, w_post[k]);
                if (FEATURE) get<VEC>(kept + (POST ? 2 : 1) * apart + i, w_gate[k]);
            }
            load(u, i, uh[k]);
            float gv[VEC], dg[VEC];
            if constexpr (FULL) load(g, i, gv);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if (POST) uh[k][j] *= rho_u;
                const float value = POST ? uh[k][j] * w_post[k][j] : uh[k][j];
                if (FULL) dg[j] = t[k][j] * value;
                if (FEATURE) sum_gate[k][j] = fmaf(t[k][j], value, sum_gate[k][j]);
                if (GATE == B2_GATE_ROW) dots[1] = fmaf(t[k][j], value, dots[1]);
                if (GATE != B2_GATE_NONE) t[k][j] *= FULL ? gv[j] : FEATURE ? w_gate[k][j] : row_gate;
                if (POST) {
                    sum_post[k][j] = fmaf(t[k][j], uh[k][j], sum_post[k][j]);
                    t[k][j] *= w_post[k][j];
                    dots[0] = fmaf(t[k][j], uh[k][j], dots[0]);
                }
            }
            if (FULL && d.d_gate) store(d.d_gate + row * d.d_gate_stride, i, dg);
        }
        if constexpr (GATE == B2_GATE_ROW) {
            cta_sums(dots, sums, turn);
        } else if constexpr (POST) {
            float one[1] = {dots[0]};
            cta_sums(one, sums, turn);
            dots[0] = one[0];
        } else {
            __syncthreads();
        }
        if (tid == 0 && next < a.rows && waits.ran_out < 2) fetch_then(next, s);
        if (GATE == B2_GATE_ROW && d.d_gate && tid == 0) d.d_gate[row] = dots[1];
        if (U && d.d_block) {
            const float mean = POST ? dots[0] * over : 0.0f;
#pragma unroll
            for (int k = 0; k < IT; ++k) {
                const int i = i0 + k * 32 * VEC;
                if (i >= F) continue;
                float v[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = POST ? rho_u * fmaf(uh[k][j], -mean, t[k][j]) : t[k][j];
                store(d.d_block + row * d.d_block_stride, i, v);
            }
        }
        if (++s == ring.stages) {
            s = 0;
            phase ^= 1;
        }
    }
    float* mine = out_sums + (long long)blockIdx.x * 3 * F;
#pragma unroll
    for (int k = 0; k < IT; ++k) {
        const int i = i0 + k * 32 * VEC;
        if (i >= F) continue;
        if (RAGGED) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if (i + j < 0 || i + j >= F) continue;
                if (d.d_pre_weight) mine[i + j] = sum_pre[k][j];
                if (POST && d.d_post_weight) mine[F + i + j] = sum_post[k][j];
                if (FEATURE && d.d_gate) mine[2 * F + i + j] = sum_gate[k][j];
            }
        } else {
            if (d.d_pre_weight) put<VEC>(mine + i, sum_pre[k]);
            if (POST && d.d_post_weight) put<VEC>(mine + F + i, sum_post[k]);
            if (FEATURE && d.d_gate) put<VEC>(mine + 2 * F + i, sum_gate[k]);
        }
    }
    __syncthreads();
    if (waits.ran_out) spoil_rows(a, d, mine, waits, ring.stages, has_ds || U);
}

// Rows of any length and alignment: a CTA adds its rows into sums of its own, [CTAs][3][F] of scratch.
template <int VEC>
__global__ void __launch_bounds__(kThreads)
norm_grad_any_kernel(const b2_norm a, const b2_norm_grads d, float* __restrict__ sums) {
    __shared__ float words[32];
    after_earlier_kernels();
    const int F = a.features;
    float* pre = sums + (long long)blockIdx.x * 3 * F;
    float* post = pre + F;
    float* gate = post + F;
    for (int i = threadIdx.x; i < 3 * F; i += kThreads) pre[i] = 0.0f;
    __syncthreads();
    auto add = [&](float* to, int i, const float* v) {
        float o[VEC];
        get<VEC>(to + i, o);
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] += v[j];
        put<VEC>(to + i, o);
    };
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float* x = a.block ? a.stream + row * a.stream_stride : a.residual + row * a.residual_stride;
        const float* u = a.block ? a.block + row * a.block_stride : nullptr;
        const float* dy = d.d_out ? d.d_out + row * d.d_out_stride : nullptr;
        const float* ds = d.d_stream ? d.d_stream + row * d.d_stream_stride : nullptr;
        const float rho = dy ? a.stream_rstd[row] : 0.0f, rho_u = a.post_weight ? a.block_rstd[row] : 1.0f;
        float mean = 0.0f;
        if (dy) {
            float q = 0.0f;
            for (int i = threadIdx.x * VEC; i < F; i += kThreads * VEC) {
                float xv[VEC], yv[VEC];
                get<VEC>(x + i, xv);
                get<VEC>(dy + i, yv);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    xv[j] *= rho;
                    q = fmaf(yv[j] * a.pre_weight[i + j], xv[j], q);
                    xv[j] *= yv[j];
                }
                add(pre, i, xv);
            }
            mean = block_sum(q, words) / (float)F;
        }
        float dot = 0.0f, dgate = 0.0f;
        for (int i = threadIdx.x * VEC; i < F; i += kThreads * VEC) {
            float t[VEC] = {}, v[VEC], g[VEC];
            if (ds) get<VEC>(ds + i, t);
            if (dy) {
                float xv[VEC], yv[VEC];
                get<VEC>(x + i, xv);
                get<VEC>(dy + i, yv);
#pragma unroll
                for (int j = 0; j < VEC; ++j) t[j] += rho * (yv[j] * a.pre_weight[i + j] - xv[j] * rho * mean);
            }
            if (d.d_residual) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = a.residual_scale * t[j];
                put<VEC>(d.d_residual + row * d.d_residual_stride + i, v);
            }
            if (!u) continue;
            get<VEC>(u + i, v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                v[j] *= rho_u;
                const float w = a.post_weight ? a.post_weight[i + j] : 1.0f;
                g[j] = t[j] * (v[j] * w);
                dgate += g[j];
                t[j] *= gate_at(a, row, i + j);
                v[j] *= t[j];
                dot = fmaf(v[j], w, dot);
            }
            if (a.gate_kind == B2_GATE_FEATURE) add(gate, i, g);
            else if (a.gate_kind == B2_GATE_FULL && d.d_gate) put<VEC>(d.d_gate + row * d.d_gate_stride + i, g);
            if (a.post_weight) add(post, i, v);
            if (d.d_block) put<VEC>(d.d_block + row * d.d_block_stride + i, t);
        }
        if (a.gate_kind == B2_GATE_ROW) {
            dgate = block_sum(dgate, words);
            if (d.d_gate && threadIdx.x == 0) d.d_gate[row] = dgate;
        }
        if (a.post_weight) {
            mean = block_sum(dot, words) / (float)F;
            if (d.d_block)
                for (int i = threadIdx.x * VEC; i < F; i += kThreads * VEC) {
                    float t[VEC], v[VEC];
                    get<VEC>(d.d_block + row * d.d_block_stride + i, t);
                    get<VEC>(u + i, v);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) t[j] = rho_u * (t[j] * a.post_weight[i + j] - v[j] * rho_u * mean);
                    put<VEC>(d.d_block + row * d.d_block_stride + i, t);
                }
        }
    }
}

// The CTAs' sums: COLS columns to a block of 1024 threads, which take the CTAs by turns.
template <int COLS>
__global__ void __launch_bounds__(1024)
norm_sums_kernel(const float* __restrict__ sums, int ctas, int F, float* pre, float* post, float* gate) {
    constexpr int TURNS = 1024 / COLS;
    __shared__ float words[TURNS][COLS + 1];
    after_earlier_kernels();
    const int col = threadIdx.x % COLS, turn = threadIdx.x / COLS;
    const int i = blockIdx.x * COLS + col;
    float* out = blockIdx.y == 0 ? pre : blockIdx.y == 1 ? post : gate;
    if (!out) return;
    float s = 0.0f;
    if (i < F)
#pragma unroll 8
        for (int c = turn; c < ctas; c += TURNS) s += sums[((long long)c * 3 + blockIdx.y) * F + i];
    words[turn][col] = s;
    __syncthreads();
    // (a warp to a column at a time)
    for (int k = threadIdx.x / 32; k < COLS && blockIdx.x * COLS + k < F; k += 32) {
        s = 0.0f;
        for (int t = threadIdx.x % 32; t < TURNS; t += 32) s += words[t][k];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (threadIdx.x % 32 == 0) out[blockIdx.x * COLS + k] = s;
    }
}

// Threads of a CTA that holds `each` values of a row to a thread; 0 where a row has too many for `most`.
int threads_of(int F, int each, int most) {
    const int t = ((F + each - 1) / each + 31) / 32 * 32;
    return t <= most ? t : 0;
}

// How the gradient is launched: eight values of a row to a thread, and CTAs for as many threads an SM as have registers
// enough, 640 (16384 rows of 1536 features: 119 us with 512, 99; of 2047: 241 and 160; of 2048, 512 in both: 127; for 768
// or 1024 none are left: 125, 151 and 141).  Two CTAs of more than 320 threads there are only without a block, whose
// gradient holds less: 1024 threads (6000 x 3501 80 and 59 us; 16384 x 2048 99 and 83).  With a block short rows take 512:
// more CTAs leave more sums (8000 x 1001 44 us, 48 with 640; without a block 16384 x 1001 61 and 48), and a gate for every
// value takes room for rows ahead (16384 x 1536 124 and 146).  Three rows ahead where they fit.
// Of rows beyond 5120 features sixteen values to a thread, whose weights lie in shared memory, read from there in every
// row: 4096 x 8192 131 us, 154 with eight values to 1024 threads and weights from L2, 144 with those in shared memory (64
// registers a thread); a gate for every value 185 and 176, which leaves shared memory for one row at a time.  Of
// 5000 features 71 us for 3000 rows, 67 with eight.
struct GradPlan {
    int threads, ctas, each, most, room;             // `most`: threads an SM that registers are shared out for
    Ring ring;
};
GradPlan grad_plan(const b2_norm& a, int tensors, bool ragged) {
    GradPlan p = {};
    const int values = a.features + (ragged ? 3 : 0);
    p.each = 8;
    p.threads = threads_of(values, 8, 640);
    if (!p.threads) {
        p.each = 16;
        p.threads = threads_of(values, 16, 512);
    }
    long long per_sm = p.threads ? 1 : 4;
    p.most = 512;
    if (p.threads && p.each == 8) {
        const int short_row = !a.block ? 0 : a.gate_kind == B2_GATE_FULL ? 256 : 128;
        const int total = !a.block && p.threads > 640 / 3 && p.threads <= 512 ? 1024 : p.threads <= short_row ? 512 : 640;
        per_sm = total / p.threads > 16 ? 16 : total / p.threads;
        p.most = per_sm * p.threads <= 512 ? 512 : per_sm * p.threads <= 640 ? 640 : 1024;
    }
    p.ctas = (int)(a.rows < b2::kSms * per_sm ? a.rows : b2::kSms * per_sm);
    if (!p.threads || !tensors) return p;
    p.ring.slot = (values + 3) / 4 * 16;
    const int weights = p.each == 16 ? 1 + (a.post_weight != nullptr) + (a.gate_kind == B2_GATE_FEATURE) : 0;
    const int room = p.each == 16 ? kGradShared - weights * p.ring.slot : (int)((220 << 10) / per_sm) - 1024;
    p.ring.stages = room / (p.ring.slot * tensors);
    if (p.ring.stages > kStages) p.ring.stages = kStages;
    if (p.ring.stages < 1) p.threads = 0;
    p.room = p.ring.slot * (weights + p.ring.stages * tensors);
    return p;
}

int check_norm(const b2_norm* a) {
    B2_REQUIRE(a, "missing argument");
    B2_REQUIRE(a->rows >= 0 && a->rows <= (1ll << 38) && a->features > 0 && a->features <= (1 << 24), "bad norm: %lld rows of %d features", (long long)a->rows, a->features);
    B2_REQUIRE(a->gate_kind >= B2_GATE_NONE && a->gate_kind <= B2_GATE_FULL, "unknown kind of gate: %d", a->gate_kind);
    B2_REQUIRE((a->gate_kind == B2_GATE_NONE) == (a->gate == nullptr), "a gate and its kind go together");
    for (const float* p : {a->block, a->residual, a->gate, a->post_weight, a->pre_weight, (const float*)a->stream, (const float*)a->out,
                           (const float*)a->block_rstd, (const float*)a->stream_rstd})
        B2_REQUIRE(((uintptr_t)p & 3) == 0, "a tensor of the norm lies between two addresses");
    if (!a->block) B2_REQUIRE(!a->gate && !a->post_weight && a->residual_scale == 1.0f, "a gate, a weight or a scale without a block");
    return B2_OK;
}

int check_stride(const b2_norm* a, const void* p, int64_t stride, const char* what) {
    B2_REQUIRE(!p || a->rows <= 1 || stride >= a->features, "rows of the %s overlap: stride %lld, %d features", what, (long long)stride, a->features);
    B2_REQUIRE(!p || a->rows <= 1 || stride <= (1ll << 46) / a->rows, "%lld rows of the %s have no memory: stride %lld", (long long)a->rows, what,
               (long long)stride);
    return B2_OK;
}

inline Rows gate_rows(const b2_norm& a, const float* p, long long stride) {
    const long long R = a.rows, F = a.features;
    return a.gate_kind == B2_GATE_FULL ? rows_at(p, R, F, stride) : a.gate_kind == B2_GATE_ROW ? rows_at(p, 1, R, R) : rows_at(p, 1, F, F);
}

int check_in_place(const b2_norm* a, const void* result, int64_t result_stride, const void* operand, int64_t stride, const char* what) {
    B2_REQUIRE(!result || result != operand || a->rows <= 1 || result_stride == stride, "%s in place of its operand has other strides: %lld, %lld", what,
               (long long)result_stride, (long long)stride);
    return B2_OK;
}

bool rows_aligned(const void* p, int64_t stride) { return b2::aligned16(p) && stride % 4 == 0; }

template <int IT, bool RAGGED>
int launch_rows(const b2_norm& a, int threads, cudaStream_t st) {
    // CTAs that go through several rows: ragged ones (148 and so every multiple of it is a multiple of four), and of up to
    // 64 threads, since a CTA to a row is bound by their start, 1.1 ns each (16384 x 64: 18 us and 10; x 256: 20 and 15)
    const int per_sm = !RAGGED || threads <= 32 ? 32 : threads > 512 ? 1 : 1024 / threads;
    const long long most = RAGGED || threads <= 64 ? (long long)b2::kSms * per_sm : 1ll << 30;
    const unsigned blocks = (unsigned)(a.rows < most ? a.rows : most);
    const size_t room = RAGGED ? (size_t)3 * ((a.features + 6) / 4 * 4) * sizeof(float) : 0;
#define B2_LAUNCH(U, POST, GATE)                                                                                                       \
    do {                                                                                                                              \
        static std::atomic<unsigned long long> done{0};                                                                               \
        if (room > 40 << 10) B2_CHECK(b2::allow_shared((const void*)norm_row_kernel<IT, RAGGED, U, POST, GATE>, 220 << 10, &done)); \
        B2_CUDA((b2::launch_after(norm_row_kernel<IT, RAGGED, U, POST, GATE>, dim3(blocks), threads, room, st, a)));              \
    } while (0)
#define B2_GATED(POST)                                                        \
    switch (a.gate_kind) {                                                    \
        case B2_GATE_FEATURE: B2_LAUNCH(true, POST, B2_GATE_FEATURE); break;  \
        case B2_GATE_ROW: B2_LAUNCH(true, POST, B2_GATE_ROW); break;          \
        case B2_GATE_FULL: B2_LAUNCH(true, POST, B2_GATE_FULL); break;        \
        default: B2_LAUNCH(true, POST, B2_GATE_NONE);                         \
    }
    if (!a.block) B2_LAUNCH(false, false, B2_GATE_NONE);
    else if (a.post_weight) B2_GATED(true)
    else B2_GATED(false)
#undef B2_GATED
#undef B2_LAUNCH
    return B2_OK;
}

template <bool RAGGED, int MOST, int IT, bool U, bool POST, int GATE>
int launch_grad(const b2_norm& a, const b2_norm_grads& d, const GradPlan& p, float* sums, cudaStream_t st) {
    static std::atomic<unsigned long long> done{0};
    B2_CHECK(b2::allow_shared((const void*)norm_grad_row_kernel<RAGGED, MOST, IT, U, POST, GATE>, kGradShared, &done));
    B2_CUDA((b2::launch_after(norm_grad_row_kernel<RAGGED, MOST, IT, U, POST, GATE>, dim3(p.ctas), p.threads, (size_t)p.room, st, a, d,
                              sums, p.ring)));
    return B2_OK;
}

template <bool RAGGED, int MOST, int IT>
int launch_grad_of(const b2_norm& a, const b2_norm_grads& d, const GradPlan& p, float* sums, cudaStream_t st) {
    if (!a.block) return launch_grad<RAGGED, MOST, IT, false, false, B2_GATE_NONE>(a, d, p, sums, st);
#define B2_GATED(POST)                                                                                               \
    switch (a.gate_kind) {                                                                                           \
        case B2_GATE_FEATURE: return launch_grad<RAGGED, MOST, IT, true, POST, B2_GATE_FEATURE>(a, d, p, sums, st);  \
        case B2_GATE_ROW: return launch_grad<RAGGED, MOST, IT, true, POST, B2_GATE_ROW>(a, d, p, sums, st);          \
        case B2_GATE_FULL: return launch_grad<RAGGED, MOST, IT, true, POST, B2_GATE_FULL>(a, d, p, sums, st);        \
        default: return launch_grad<RAGGED, MOST, IT, true, POST, B2_GATE_NONE>(a, d, p, sums, st);                  \
    }
    if (a.post_weight) B2_GATED(true)
    B2_GATED(false)
#undef B2_GATED
}

}  // namespace

extern "C" int b2_norm_fprop(const b2_norm* a, void* stream) {
    B2_CHECK(check_norm(a));
    B2_REQUIRE((a->out != nullptr) == (a->pre_weight != nullptr), "out and pre_weight go together");
    B2_REQUIRE(a->block || a->out, "nothing to compute");
    B2_REQUIRE((a->block != nullptr) == (a->stream != nullptr), "the stream is stored where there is a block");
    if (a->rows == 0) return B2_OK;
    B2_REQUIRE(a->residual, "missing residual");
    B2_CHECK(check_stride(a, a->block, a->block_stride, "block"));
    B2_CHECK(check_stride(a, a->residual, a->residual_stride, "residual"));
    B2_CHECK(check_stride(a, a->stream, a->stream_stride, "stream"));
    B2_CHECK(check_stride(a, a->out, a->out_stride, "result"));
    if (a->gate_kind == B2_GATE_FULL) B2_CHECK(check_stride(a, a->gate, a->gate_stride, "gate"));
    const long long R = a->rows, F = a->features;
    const Rows results[] = {rows_at(a->out, R, F, a->out_stride), rows_at(a->stream, R, F, a->stream_stride), rows_at(a->block_rstd, 1, R, R),
                            rows_at(a->stream_rstd, 1, R, R)};
    const Rows operands[] = {rows_at(a->block, R, F, a->block_stride), gate_rows(*a, a->gate, a->gate_stride), rows_at(a->post_weight, 1, F, F),
                             rows_at(a->pre_weight, 1, F, F), rows_at(a->stream == a->residual ? nullptr : a->residual, R, F, a->residual_stride)};
    B2_CHECK(check_apart(results, 4, operands, 5, "norm"));
    B2_CHECK(check_in_place(a, a->stream, a->stream_stride, a->residual, a->residual_stride, "the stream"));
    b2::Memory memory;
    B2_CHECK(memory.find_device());
    if (a->out) B2_CHECK(memory.written(a->out, "the norm's result"));
    if (a->stream) B2_CHECK(memory.written(a->stream, "the stream"));
    for (const float* p : {a->block_rstd, a->stream_rstd})
        if (p) B2_CHECK(memory.written(p, "a reciprocal deviation of the norm"));
    for (const float* p : {a->post_weight, a->pre_weight}) B2_CHECK(memory.read(p, "a weight of the norm"));
    B2_CHECK(memory.read(a->gate, "the gate"));
    B2_CHECK(memory.read(a->residual, "the residual"));
    B2_CHECK(memory.read(a->block, "the block"));
    const unsigned blocks = (unsigned)(a->rows < (1ll << 30) ? a->rows : (1ll << 30));
    cudaStream_t st = (cudaStream_t)stream;
    const bool vec = F % 4 == 0 && rows_aligned(a->block, a->block_stride) && rows_aligned(a->residual, a->residual_stride) &&
                     rows_aligned(a->stream, a->stream_stride) && rows_aligned(a->out, a->out_stride) &&
                     (a->gate_kind != B2_GATE_FULL ? a->gate_kind == B2_GATE_ROW || b2::aligned16(a->gate) : rows_aligned(a->gate, a->gate_stride)) &&
                     b2::aligned16(a->post_weight) && b2::aligned16(a->pre_weight);
    // all rows as far behind a boundary
    auto alike = [&](const float* p, int64_t stride) {
        return !p || (shift_of(p) == shift_of(a->residual) && (a->rows <= 1 || (stride - a->residual_stride) % 4 == 0));
    };
    // (rows fetched ahead are device memory)
    const bool ragged = !memory.elsewhere && alike(a->block, a->block_stride) && alike(a->stream, a->stream_stride) && alike(a->out, a->out_stride) &&
                        (a->gate_kind != B2_GATE_FULL || alike(a->gate, a->gate_stride));
    // Few rows: as many threads as a row has vectors, for the least latency.  Many: eight values to a thread, sixteen from
    // 2048 features on, so that several rows share an SM and the sums over the CTA weigh less (8192 x 4096: 100 us
    // with eight, 85 with sixteen; 16384 x 512: 25 and 27).
    const bool few = a->rows <= b2::kSms * 2, wide = F >= 2048;
#define B2_ROWS(IT, RAGGED) \
    if (const int t = threads_of(F + (RAGGED ? 3 : 0), 4 * IT, 1024)) return launch_rows<IT, RAGGED>(*a, t, st);
    if (vec) {
        if (few) B2_ROWS(1, false)
        if (!wide) B2_ROWS(2, false)
        B2_ROWS(4, false)
    } else if (ragged) {
        if (few) B2_ROWS(1, true)
        if (!wide) B2_ROWS(2, true)
        B2_ROWS(4, true)
    }
#undef B2_ROWS
    B2_CUDA(b2::launch_after(vec ? norm_any_kernel<4> : norm_any_kernel<1>, dim3(blocks), kThreads, 0, st, *a));
    return B2_OK;
}

extern "C" int b2_norm_bprop_scratch_bytes(const b2_norm* a, size_t* bytes) {
    B2_REQUIRE(bytes, "missing argument");
    B2_CHECK(check_norm(a));
    const int even = grad_plan(*a, 1, false).ctas, ragged = grad_plan(*a, 1, true).ctas;        // (they do not depend on the tensors)
    *bytes = (size_t)(even > ragged ? even : ragged) * 3 * a->features * sizeof(float) + 256;
    return B2_OK;
}

extern "C" int b2_norm_bprop(const b2_norm* a, const b2_norm_grads* d, void* scratch, size_t scratch_bytes, void* stream) {
    size_t need = 0;
    B2_CHECK(b2_norm_bprop_scratch_bytes(a, &need));
    B2_REQUIRE(d, "missing argument");
    for (const float* p : {d->d_out, d->d_stream, (const float*)d->d_residual, (const float*)d->d_block, (const float*)d->d_gate,
                           (const float*)d->d_post_weight, (const float*)d->d_pre_weight})
        B2_REQUIRE(((uintptr_t)p & 3) == 0, "a gradient of the norm lies between two addresses");
    B2_REQUIRE(((uintptr_t)d->status & 3) == 0, "the status lies between two addresses");
    B2_REQUIRE(scratch && scratch_bytes >= need, "the norm's gradient needs %zu bytes of scratch, got %zu", need, scratch_bytes);
    const Rows room = rows_at((const float*)(((uintptr_t)scratch + 3) / 4 * 4), 1, (long long)(need / 4), (long long)(need / 4));     // (the sums of CTAs)
    B2_REQUIRE(a->pre_weight ? d->d_out != nullptr || a->rows == 0 : d->d_out == nullptr && d->d_pre_weight == nullptr, "d_out and pre_weight go together");
    B2_REQUIRE(a->pre_weight || d->d_stream || a->rows == 0, "no gradient to start from");
    B2_REQUIRE(a->block || (!d->d_block && !d->d_gate), "gradients of a block that is not there");
    B2_REQUIRE(a->gate || !d->d_gate, "the gradient of a gate that is not there");
    B2_REQUIRE(a->post_weight || !d->d_post_weight, "the gradient of a weight that is not there");
    if (a->rows > 0) {
        B2_REQUIRE(!a->pre_weight || (a->stream_rstd && (a->block ? a->stream : a->residual)), "the gradient reads the stream and its stream_rstd");
        B2_REQUIRE(!a->post_weight || a->block_rstd, "the gradient reads block_rstd");
        B2_CHECK(check_stride(a, a->block, a->block_stride, "block"));
        if (a->block) B2_CHECK(check_stride(a, a->stream, a->stream_stride, "stream"));
        else B2_CHECK(check_stride(a, a->residual, a->residual_stride, "residual"));
        if (a->gate_kind == B2_GATE_FULL) B2_CHECK(check_stride(a, a->gate, a->gate_stride, "gate"));
        B2_CHECK(check_stride(a, d->d_out, d->d_out_stride, "result's gradient"));
        B2_CHECK(check_stride(a, d->d_stream, d->d_stream_stride, "stream's gradient"));
        B2_CHECK(check_stride(a, d->d_residual, d->d_residual_stride, "residual's gradient"));
        B2_CHECK(check_stride(a, d->d_block, d->d_block_stride, "block's gradient"));
        if (a->gate_kind == B2_GATE_FULL) B2_CHECK(check_stride(a, d->d_gate, d->d_gate_stride, "gate's gradient"));
        const long long R = a->rows, F = a->features;
        const Rows results[] = {rows_at(d->d_residual, R, F, d->d_residual_stride), rows_at(d->d_block, R, F, d->d_block_stride),
                                gate_rows(*a, d->d_gate, d->d_gate_stride), rows_at(d->d_post_weight, 1, F, F), rows_at(d->d_pre_weight, 1, F, F), room};
        const Rows operands[] = {a->block ? rows_at(a->stream, R, F, a->stream_stride) : rows_at(a->residual, R, F, a->residual_stride),
                                 rows_at(a->block, R, F, a->block_stride), gate_rows(*a, a->gate, a->gate_stride), rows_at(a->post_weight, 1, F, F),
                                 rows_at(a->pre_weight, 1, F, F), rows_at(d->d_out, R, F, d->d_out_stride), rows_at(a->stream_rstd, 1, R, R),
                                 rows_at(a->block_rstd, 1, R, R), rows_at(d->d_stream == d->d_residual ? nullptr : d->d_stream, R, F, d->d_stream_stride)};
        B2_CHECK(check_apart(results, 6, operands, 9, "norm"));
        B2_CHECK(check_in_place(a, d->d_residual, d->d_residual_stride, d->d_stream, d->d_stream_stride, "the residual's gradient"));
    }
    // (sums over rows are written whatever the number of rows)
    float* gate = a->gate_kind == B2_GATE_FEATURE ? d->d_gate : nullptr;
    if (a->rows == 0) {
        const long long F = a->features;
        const Rows results[] = {rows_at(d->d_post_weight, 1, F, F), rows_at(d->d_pre_weight, 1, F, F), rows_at(gate, 1, F, F), room};
        B2_CHECK(check_apart(results, 4, nullptr, 0, "norm"));
    }
    b2::Memory memory;
    B2_CHECK(memory.find_device());
    B2_CHECK(memory.written(scratch, "the norm's scratch"));
    if (d->status) B2_CHECK(memory.written(d->status, "the status"));
    for (const float* p : {d->d_pre_weight, d->d_post_weight, gate})
        if (p) B2_CHECK(memory.written(p, "a gradient of the norm"));
    if (a->rows > 0) {
        for (const float* p : {d->d_residual, d->d_block, gate ? nullptr : d->d_gate})
            if (p) B2_CHECK(memory.written(p, "a gradient of the norm"));
        const float* read[] = {a->block ? a->stream : a->residual, a->block, a->gate, a->post_weight, a->pre_weight,
                               a->post_weight ? a->block_rstd : nullptr, a->pre_weight ? a->stream_rstd : nullptr, d->d_out, d->d_stream};
        for (const float* p : read) B2_CHECK(memory.read(p, "an operand of the norm's gradient"));
    }
    cudaStream_t st = (cudaStream_t)stream;
    float* sums = (float*)(((uintptr_t)scratch + 255) / 256 * 256);
    const bool full = a->gate_kind == B2_GATE_FULL;
    const int tensors = (d->d_out ? 2 : 0) + (d->d_stream ? 1 : 0) + (a->block ? 1 : 0) + (full ? 1 : 0);
    const float* x = a->block ? a->stream : a->residual;
    const int64_t x_stride = a->block ? a->stream_stride : a->residual_stride;
    const bool vec = a->features % 4 == 0 && rows_aligned(a->block, a->block_stride) && (!d->d_out || rows_aligned(x, x_stride)) &&
                     rows_aligned(d->d_out, d->d_out_stride) && rows_aligned(d->d_stream, d->d_stream_stride) &&
                     rows_aligned(d->d_residual, d->d_residual_stride) && rows_aligned(d->d_block, d->d_block_stride) &&
                     (full ? rows_aligned(a->gate, a->gate_stride) && rows_aligned(d->d_gate, d->d_gate_stride) : a->gate_kind == B2_GATE_ROW || b2::aligned16(a->gate)) &&
                     b2::aligned16(a->post_weight) && b2::aligned16(a->pre_weight);
    auto alike = [&](const float* q, int64_t stride) {
        return !q || (shift_of(q) == shift_of(x) && (a->rows <= 1 || (stride - x_stride) % 4 == 0));
    };
    const bool ragged = !vec && alike(a->block, a->block_stride) && alike(d->d_out, d->d_out_stride) && alike(d->d_stream, d->d_stream_stride) &&
                        alike(d->d_residual, d->d_residual_stride) && alike(d->d_block, d->d_block_stride) &&
                        (!full || (alike(a->gate, a->gate_stride) && alike(d->d_gate, d->d_gate_stride)));
    const GradPlan p = grad_plan(*a, tensors, ragged);
    if (p.ctas > 0) {
        // (bulk copies are from device memory alone)
        if (!p.threads || !d->d_out || memory.elsewhere || !(vec || ragged)) B2_CUDA(b2::launch_after(vec ? norm_grad_any_kernel<4> : norm_grad_any_kernel<1>, dim3(p.ctas), kThreads, 0, st, *a, *d, sums));
#define B2_GRAD(MOST, EACH)                                                                                  \
    else if (p.most == MOST && p.each == EACH) {                                                             \
        if (vec) B2_CHECK((launch_grad_of<false, MOST, EACH / 4>(*a, *d, p, sums, st)));            \
        else B2_CHECK((launch_grad_of<true, MOST, EACH / 4>(*a, *d, p, sums, st)));                 \
    }
        B2_GRAD(512, 8)
        B2_GRAD(640, 8)
        B2_GRAD(512, 16)
        else if (vec) B2_CHECK((launch_grad<false, 1024, 2, false, false, B2_GATE_NONE>(*a, *d, p, sums, st)));
        else B2_CHECK((launch_grad<true, 1024, 2, false, false, B2_GATE_NONE>(*a, *d, p, sums, st)));
#undef B2_GRAD
    }
    if (d->d_pre_weight || d->d_post_weight || gate)
    {
        // (many CTAs' sums of few columns: fewer columns to a block)
        const bool narrow = p.ctas > 512;
        const int cols = narrow ? 8 : 32;
        B2_CUDA(b2::launch_after(narrow ? norm_sums_kernel<8> : norm_sums_kernel<32>, dim3((a->features + cols - 1) / cols, 3), 1024, 0, st,
                                 (const float*)sums, p.ctas, a->features, d->d_pre_weight, d->d_post_weight, gate));
    }
    return B2_OK;
}
