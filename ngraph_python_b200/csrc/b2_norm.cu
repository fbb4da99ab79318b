// The edge between two blocks of a residual network, and its gradients:
//
//   stream = a residual + gate * (rms(block) * w_post),   out = rms(stream) * w_pre,   rms(x) = x * rstd(x)
//
//   d_stream' = d_stream + through(d_out, stream, w_pre),  d_residual = a d_stream',  d_gate = d_stream' * rms(block) w_post
//   d_block   = through(gate * d_stream', block, w_post)
//   through(d, x, w) = rstd (w d - x^ mean(w d x^)),  x^ = x rstd;   d_w = sum over rows of d x^
#include <cstdint>

#include "b2_operators.h"
#include "b2_ew_device.cuh"

namespace {

constexpr int kThreads = 256;

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

// Sums of two values over the CTA, the same bits in every thread.  One barrier: calls write to two sets of words by
// turns, and who comes to write to a set again has passed the barrier behind which everybody had read it.
struct TwoSums {
    float words[2][2][32];
};
__device__ __forceinline__ void cta_sums(float& x, float& y, TwoSums& s, int& turn) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        x += __shfl_xor_sync(0xffffffffu, x, o);
        y += __shfl_xor_sync(0xffffffffu, y, o);
    }
    if (lane == 0) {
        s.words[turn][0][warp] = x;
        s.words[turn][1][warp] = y;
    }
    __syncthreads();
    x = lane < warps ? s.words[turn][0][lane] : 0.0f;
    y = lane < warps ? s.words[turn][1][lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        x += __shfl_xor_sync(0xffffffffu, x, o);
        y += __shfl_xor_sync(0xffffffffu, y, o);
    }
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

__device__ __forceinline__ float rstd_of(float squares, int F, float eps) { return 1.0f / sqrtf(squares / (float)F + eps); }

__device__ __forceinline__ float gate_at(const b2_norm& a, long long row, int i) {
    switch (a.gate_kind) {
        case B2_GATE_FEATURE: return a.gate[i];
        case B2_GATE_ROW: return a.gate[row];
        case B2_GATE_FULL: return a.gate[row * a.gate_stride + i];
        default: return 1.0f;
    }
}

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
            for (int i = threadIdx.x; i < F; i += kThreads) q += u[i] * u[i];
            rho = rstd_of(block_sum(q, words), F, a.eps);
            if (a.block_rstd && threadIdx.x == 0) a.block_rstd[row] = rho;
        }
        float q = 0.0f;
        for (int i = threadIdx.x; i < F; i += kThreads) {
            float x = r[i];
            if (u) {
                float y = u[i];
                if (a.post_weight) y = y * rho * a.post_weight[i];
                x = a.residual_scale * x + y * gate_at(a, row, i);
                s[i] = x;
            }
            q += x * x;
        }
        if (!a.out && !a.stream_rstd) continue;
        rho = rstd_of(block_sum(q, words), F, a.eps);
        if (a.stream_rstd && threadIdx.x == 0) a.stream_rstd[row] = rho;
        if (a.out)
            for (int i = threadIdx.x; i < F; i += kThreads) a.out[row * a.out_stride + i] = (s ? s[i] : r[i]) * rho * a.pre_weight[i];
    }
}

// A row to a CTA, held in registers: each tensor is read once.  Both operands are on their way before the first sum.
template <int VEC, int IT>
__global__ void __launch_bounds__(1024)
norm_row_kernel(const b2_norm a) {
    __shared__ TwoSums sums;
    after_earlier_kernels();
    const int F = a.features, T = blockDim.x;
    int turn = 0;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float x[IT][VEC] = {}, u[IT][VEC] = {};
        const float* r = a.residual + row * a.residual_stride;
        const float* b = a.block ? a.block + row * a.block_stride : nullptr;
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const int i = (k * T + threadIdx.x) * VEC;
            if (i < F) {
                if (b) get<VEC>(b + i, u[k]);
                get<VEC>(r + i, x[k]);
            }
        }
        if (b) {
            float rho = 1.0f;
            if (a.post_weight) {
                float q = 0.0f, none = 0.0f;
#pragma unroll
                for (int k = 0; k < IT; ++k)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) q += u[k][j] * u[k][j];
                cta_sums(q, none, sums, turn);
                rho = rstd_of(q, F, a.eps);
                if (a.block_rstd && threadIdx.x == 0) a.block_rstd[row] = rho;
            }
            const float row_gate = a.gate_kind == B2_GATE_ROW ? a.gate[row] : 1.0f;
            const float* g = a.gate_kind == B2_GATE_FEATURE ? a.gate : a.gate_kind == B2_GATE_FULL ? a.gate + row * a.gate_stride : nullptr;
            float* s = a.stream + row * a.stream_stride;
#pragma unroll
            for (int k = 0; k < IT; ++k) {
                const int i = (k * T + threadIdx.x) * VEC;
                if (i < F) {
                    float w[VEC], gv[VEC];
                    if (a.post_weight) get<VEC>(a.post_weight + i, w);
                    if (g) get<VEC>(g + i, gv);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        float y = u[k][j];
                        if (a.post_weight) y = y * rho * w[j];
                        y = y * (g ? gv[j] : row_gate);
                        x[k][j] = a.residual_scale * x[k][j] + y;
                    }
                    put<VEC>(s + i, x[k]);
                }
            }
        }
        if (!a.out && !a.stream_rstd) continue;
        float q = 0.0f, none = 0.0f;
#pragma unroll
        for (int k = 0; k < IT; ++k)
#pragma unroll
            for (int j = 0; j < VEC; ++j) q += x[k][j] * x[k][j];
        cta_sums(q, none, sums, turn);
        const float rho = rstd_of(q, F, a.eps);
        if (a.stream_rstd && threadIdx.x == 0) a.stream_rstd[row] = rho;
        if (!a.out) continue;
        float* o = a.out + row * a.out_stride;
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const int i = (k * T + threadIdx.x) * VEC;
            if (i < F) {
                float w[VEC];
                get<VEC>(a.pre_weight + i, w);
#pragma unroll
                for (int j = 0; j < VEC; ++j) w[j] = x[k][j] * rho * w[j];
                put<VEC>(o + i, w);
            }
        }
    }
}

// Gradients, a row to a CTA at a time.  A CTA keeps its rows' sums for the weights and a gate per feature in registers.
// The tensors of its next rows are on their way into shared memory meanwhile (bulk copies; a ring of `stages` rows),
// since between the loads of a row and its stores there are two sums over the CTA: the first pair (stream, d_out) of a
// place is free again behind the first of them, the others behind the second.  Rows of any alignment: a copy starts at
// the 16-byte boundary below the row.  A wait that runs out turns the results into NaN.
constexpr int kStages = 4;

struct Ring {
    int stages, slot;                   // bytes of one tensor's row, with room for its alignment
};

template <int VEC, int IT>
__global__ void __launch_bounds__(512)
norm_grad_row_kernel(const b2_norm a, const b2_norm_grads d, float* __restrict__ out_sums, const Ring ring) {
    extern __shared__ __align__(128) unsigned char room[];
    __shared__ unsigned long long first_full[kStages], then_full[kStages];
    __shared__ TwoSums sums;
    constexpr bool HOLD = VEC * IT <= 8;        // weights stay in registers
    const int F = a.features, T = blockDim.x, tid = threadIdx.x;
    const bool has_dy = d.d_out != nullptr, has_ds = d.d_stream != nullptr, has_u = a.block != nullptr, post = a.post_weight != nullptr;
    const bool full_gate = a.gate_kind == B2_GATE_FULL, feature_gate = a.gate_kind == B2_GATE_FEATURE;
    // places of the tensors within a stage
    const int at_dy = ring.slot, at_ds = has_dy ? 2 * ring.slot : 0, at_u = at_ds + (has_ds ? ring.slot : 0), at_g = at_u + (has_u ? ring.slot : 0);
    const int stage_bytes = at_g + (full_gate ? ring.slot : 0);
    const float* xs = has_u ? a.stream : a.residual;
    const long long xs_stride = has_u ? a.stream_stride : a.residual_stride;
    if (tid == 0) {
        for (int s = 0; s < ring.stages; ++s) {
            b2_mbar_init(first_full + s, 1);
            b2_mbar_init(then_full + s, 1);
        }
        b2_mbar_init_fence();
    }
    __syncthreads();
    after_earlier_kernels();

    auto shift_of = [](const float* p) { return (int)(((uintptr_t)p >> 2) & 3); };
    auto bytes_of = [&](const float* p) { return (unsigned)((shift_of(p) + F + 3) / 4 * 16); };
    auto copy = [&](const float* p, int to, unsigned long long* bar) { b2_bulk_g2s(room + to, p - shift_of(p), bytes_of(p), bar); };
    auto fetch_first = [&](long long row, int s) {
        if (!has_dy) return;
        const float *x = xs + row * xs_stride, *dy = d.d_out + row * d.d_out_stride;
        b2_mbar_expect_tx(first_full + s, bytes_of(x) + bytes_of(dy));
        copy(x, s * stage_bytes, first_full + s);
        copy(dy, s * stage_bytes + at_dy, first_full + s);
    };
    auto fetch_then = [&](long long row, int s) {
        const float *ds = has_ds ? d.d_stream + row * d.d_stream_stride : nullptr, *u = has_u ? a.block + row * a.block_stride : nullptr,
                    *g = full_gate ? a.gate + row * a.gate_stride : nullptr;
        if (!ds && !u && !g) return;
        b2_mbar_expect_tx(then_full + s, (ds ? bytes_of(ds) : 0u) + (u ? bytes_of(u) : 0u) + (g ? bytes_of(g) : 0u));
        if (ds) copy(ds, s * stage_bytes + at_ds, then_full + s);
        if (u) copy(u, s * stage_bytes + at_u, then_full + s);
        if (g) copy(g, s * stage_bytes + at_g, then_full + s);
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
    auto weights_first = [&](int k, int i) {
        if (has_dy && i < F) get<VEC>(a.pre_weight + i, w_pre[k]);
    };
    auto weights_then = [&](int k, int i) {
        if (post && i < F) get<VEC>(a.post_weight + i, w_post[k]);
        if (feature_gate && i < F) get<VEC>(a.gate + i, w_gate[k]);
    };
    if constexpr (HOLD)
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            weights_first(k, (k * T + tid) * VEC);
            weights_then(k, (k * T + tid) * VEC);
        }
    const float over = 1.0f / (float)F;
    int turn = 0, s = 0;
    unsigned phase = 0;
    bool late = false;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const long long next = row + (long long)ring.stages * gridDim.x;
        const unsigned char* here = room + s * stage_bytes;
        float t[IT][VEC] = {};
        const float rho = has_dy ? a.stream_rstd[row] : 0.0f, rho_u = post ? a.block_rstd[row] : 1.0f;
        const float row_gate = a.gate_kind == B2_GATE_ROW ? a.gate[row] : 1.0f;
        if (has_dy) {
            late |= !b2_mbar_wait(first_full + s, phase);
            const float* x = reinterpret_cast<const float*>(here) + (VEC == 4 ? 0 : shift_of(xs + row * xs_stride));
            const float* dy = reinterpret_cast<const float*>(here + at_dy) + (VEC == 4 ? 0 : shift_of(d.d_out + row * d.d_out_stride));
            float xh[IT][VEC];
            float q = 0.0f, none = 0.0f;
#pragma unroll
            for (int k = 0; k < IT; ++k) {
                const int i = (k * T + tid) * VEC;
                if constexpr (!HOLD) weights_first(k, i);
                float v[VEC] = {}, y[VEC] = {};
                if (i < F) {
                    get<VEC>(x + i, v);
                    get<VEC>(dy + i, y);
                }
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    xh[k][j] = v[j] * rho;
                    sum_pre[k][j] += y[j] * xh[k][j];
                    t[k][j] = y[j] * w_pre[k][j];
                    q += t[k][j] * xh[k][j];
                }
            }
            cta_sums(q, none, sums, turn);
            if (tid == 0 && next < a.rows) fetch_first(next, s);
            const float mean = q * over;
#pragma unroll
            for (int k = 0; k < IT; ++k)
#pragma unroll
                for (int j = 0; j < VEC; ++j) t[k][j] = rho * (t[k][j] - xh[k][j] * mean);
        }
        if (has_ds || has_u || full_gate) late |= !b2_mbar_wait(then_full + s, phase);
        const float* ds = has_ds ? reinterpret_cast<const float*>(here + at_ds) + (VEC == 4 ? 0 : shift_of(d.d_stream + row * d.d_stream_stride)) : nullptr;
        const float* u = has_u ? reinterpret_cast<const float*>(here + at_u) + (VEC == 4 ? 0 : shift_of(a.block + row * a.block_stride)) : nullptr;
        const float* g = full_gate ? reinterpret_cast<const float*>(here + at_g) + (VEC == 4 ? 0 : shift_of(a.gate + row * a.gate_stride)) : nullptr;
        float uh[IT][VEC] = {};
        float dot = 0.0f, dgate = 0.0f;
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const int i = (k * T + tid) * VEC;
            if (i >= F) continue;
            float v[VEC];
            if (ds) {
                get<VEC>(ds + i, v);
#pragma unroll
                for (int j = 0; j < VEC; ++j) t[k][j] += v[j];
            }
            if (late)
#pragma unroll
                for (int j = 0; j < VEC; ++j) t[k][j] = __int_as_float(0x7fffffff);
            if (d.d_residual) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = a.residual_scale * t[k][j];
                put<VEC>(d.d_residual + row * d.d_residual_stride + i, v);
            }
            if (!u) continue;
            if constexpr (!HOLD) weights_then(k, i);
            get<VEC>(u + i, uh[k]);
            float gv[VEC], dg[VEC];
            if (g) get<VEC>(g + i, gv);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                uh[k][j] *= rho_u;
                const float w = post ? w_post[k][j] : 1.0f;
                dg[j] = t[k][j] * (uh[k][j] * w);
                sum_gate[k][j] += dg[j];
                dgate += dg[j];
                t[k][j] *= g ? gv[j] : feature_gate ? w_gate[k][j] : row_gate;
                sum_post[k][j] += t[k][j] * uh[k][j];
                t[k][j] *= w;
                dot += t[k][j] * uh[k][j];
            }
            if (g && d.d_gate) put<VEC>(d.d_gate + row * d.d_gate_stride + i, dg);
        }
        cta_sums(dot, dgate, sums, turn);
        if (tid == 0 && next < a.rows) fetch_then(next, s);
        if (a.gate_kind == B2_GATE_ROW && d.d_gate && tid == 0) d.d_gate[row] = dgate;
        if (d.d_block) {
            const float mean = post ? dot * over : 0.0f;
#pragma unroll
            for (int k = 0; k < IT; ++k) {
                const int i = (k * T + tid) * VEC;
                if (i >= F) continue;
                float v[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = rho_u * (t[k][j] - uh[k][j] * mean);
                put<VEC>(d.d_block + row * d.d_block_stride + i, v);
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
        const int i = (k * T + tid) * VEC;
        if (i >= F) continue;
        if (d.d_pre_weight) put<VEC>(mine + i, sum_pre[k]);
        if (d.d_post_weight) put<VEC>(mine + F + i, sum_post[k]);
        if (feature_gate && d.d_gate) put<VEC>(mine + 2 * F + i, sum_gate[k]);
    }
}

// Sums over rows: a CTA adds its rows into sums of its own, [CTAs][3][F] of scratch, which norm_sums_kernel adds.
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
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float* x = a.block ? a.stream + row * a.stream_stride : a.residual + row * a.residual_stride;
        const float* u = a.block ? a.block + row * a.block_stride : nullptr;
        const float* dy = d.d_out ? d.d_out + row * d.d_out_stride : nullptr;
        const float* ds = d.d_stream ? d.d_stream + row * d.d_stream_stride : nullptr;
        const float rho = dy ? a.stream_rstd[row] : 0.0f, rho_u = a.post_weight ? a.block_rstd[row] : 1.0f;
        float mean = 0.0f;
        if (dy) {
            float q = 0.0f;
            for (int i = threadIdx.x; i < F; i += kThreads) {
                const float xh = x[i] * rho;
                q += dy[i] * a.pre_weight[i] * xh;
                pre[i] += dy[i] * xh;
            }
            mean = block_sum(q, words) / (float)F;
        }
        float dot = 0.0f, dgate = 0.0f;
        for (int i = threadIdx.x; i < F; i += kThreads) {
            float t = ds ? ds[i] : 0.0f;
            if (dy) t += rho * (dy[i] * a.pre_weight[i] - x[i] * rho * mean);
            if (d.d_residual) d.d_residual[row * d.d_residual_stride + i] = a.residual_scale * t;
            if (!u) continue;
            const float uh = u[i] * rho_u, w = a.post_weight ? a.post_weight[i] : 1.0f;
            if (a.gate_kind) {
                const float g = t * (uh * w);
                if (a.gate_kind == B2_GATE_FEATURE) gate[i] += g;
                else if (a.gate_kind == B2_GATE_ROW) dgate += g;
                else if (d.d_gate) d.d_gate[row * d.d_gate_stride + i] = g;
                t *= gate_at(a, row, i);
            }
            if (a.post_weight) {
                dot += t * w * uh;
                post[i] += t * uh;
            }
            if (d.d_block) d.d_block[row * d.d_block_stride + i] = t;
        }
        if (a.gate_kind == B2_GATE_ROW) {
            dgate = block_sum(dgate, words);
            if (d.d_gate && threadIdx.x == 0) d.d_gate[row] = dgate;
        }
        if (a.post_weight) {
            mean = block_sum(dot, words) / (float)F;
            if (d.d_block)
                for (int i = threadIdx.x; i < F; i += kThreads) {
                    float* p = d.d_block + row * d.d_block_stride + i;
                    *p = rho_u * (*p * a.post_weight[i] - u[i] * rho_u * mean);
                }
        }
    }
}

// The CTAs' sums: 32 columns to a block, whose warps take the CTAs by turns.
__global__ void __launch_bounds__(1024)
norm_sums_kernel(const float* __restrict__ sums, int ctas, int F, float* pre, float* post, float* gate) {
    __shared__ float words[32][33];
    after_earlier_kernels();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int i = blockIdx.x * 32 + lane;
    float* out = blockIdx.y == 0 ? pre : blockIdx.y == 1 ? post : gate;
    if (!out) return;
    float s = 0.0f;
    if (i < F)
#pragma unroll 4
        for (int c = warp; c < ctas; c += 32) s += sums[((long long)c * 3 + blockIdx.y) * F + i];
    words[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && i < F) {
        s = 0.0f;
        for (int w = 0; w < 32; ++w) s += words[w][lane];
        out[i] = s;
    }
}

// Threads of a CTA that holds `each` values of a row to a thread; 0 where a row has too many for `most`.
int threads_of(int F, int each, int most) {
    const int t = ((F + each - 1) / each + 31) / 32 * 32;
    return t <= most ? t : 0;
}

// How the gradient is launched: eight values to a thread, sixteen from 4096 features on (a CTA of 512 threads then
// has the registers of an SM), CTAs for about 512 threads an SM, three rows ahead where they fit.  CTAs also bound
// the sums that are left to add.
struct GradPlan {
    int threads, each, ctas;
    Ring ring;
};
GradPlan grad_plan(const b2_norm& a, int tensors) {
    GradPlan p = {};
    p.each = threads_of(a.features, 8, 512) ? 8 : 16;
    p.threads = threads_of(a.features, p.each, 512);
    long long per_sm = p.threads ? 512 / p.threads : 4;
    if (per_sm > 16) per_sm = 16;
    p.ctas = (int)(a.rows < b2::kSms * per_sm ? a.rows : b2::kSms * per_sm);
    if (!p.threads) return p;
    p.ring.slot = (a.features + 3 + 3) / 4 * 16;
    const int room = (int)((220 << 10) / per_sm) - 1024;
    p.ring.stages = room / (p.ring.slot * tensors);
    if (p.ring.stages > 3) p.ring.stages = 3;
    if (p.ring.stages < 1) p.threads = 0;
    return p;
}

int check_norm(const b2_norm* a) {
    B2_REQUIRE(a, "missing argument");
    B2_REQUIRE(a->rows >= 0 && a->features > 0 && a->features <= (1 << 24), "bad norm: %lld rows of %d features", (long long)a->rows, a->features);
    B2_REQUIRE(a->gate_kind >= B2_GATE_NONE && a->gate_kind <= B2_GATE_FULL, "unknown kind of gate: %d", a->gate_kind);
    B2_REQUIRE((a->gate_kind == B2_GATE_NONE) == (a->gate == nullptr), "a gate and its kind go together");
    if (!a->block) B2_REQUIRE(!a->gate && !a->post_weight && a->residual_scale == 1.0f, "a gate, a weight or a scale without a block");
    return B2_OK;
}

int check_stride(const b2_norm* a, const void* p, int64_t stride, const char* what) {
    B2_REQUIRE(!p || a->rows <= 1 || stride >= a->features, "rows of the %s overlap: stride %lld, %d features", what, (long long)stride, a->features);
    return B2_OK;
}

bool rows_aligned(const void* p, int64_t stride) { return b2::aligned16(p) && stride % 4 == 0; }

template <int VEC, int IT>
int launch_grad(const b2_norm& a, const b2_norm_grads& d, const GradPlan& p, int tensors, float* sums, cudaStream_t st) {
    static std::atomic<unsigned long long> done{0};
    B2_CHECK(b2::allow_shared((const void*)norm_grad_row_kernel<VEC, IT>, 220 << 10, &done));
    B2_CUDA((b2::launch_after(norm_grad_row_kernel<VEC, IT>, dim3(p.ctas), p.threads, (size_t)p.ring.stages * p.ring.slot * tensors, st, a, d, sums, p.ring)));
    return B2_OK;
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
    B2_CHECK(b2::require_here(a->out ? a->out : a->stream, "the norm's result"));
    const unsigned blocks = (unsigned)(a->rows < (1ll << 30) ? a->rows : (1ll << 30));
    const int F = a->features;
    cudaStream_t st = (cudaStream_t)stream;
    const bool vec = F % 4 == 0 && rows_aligned(a->block, a->block_stride) && rows_aligned(a->residual, a->residual_stride) &&
                     rows_aligned(a->stream, a->stream_stride) && rows_aligned(a->out, a->out_stride) &&
                     (a->gate_kind != B2_GATE_FULL ? a->gate_kind == B2_GATE_ROW || b2::aligned16(a->gate) : rows_aligned(a->gate, a->gate_stride)) &&
                     b2::aligned16(a->post_weight) && b2::aligned16(a->pre_weight);
    // few rows: as many threads as a row has vectors, for the least latency; many: eight values to a thread, so that
    // several rows share an SM
    const bool few = a->rows <= b2::kSms * 2;
#define B2_ROWS(VEC, IT)                                                                                              \
    if (const int t = threads_of(F, VEC * IT, 1024)) {                                                               \
        B2_CUDA((b2::launch_after(norm_row_kernel<VEC, IT>, dim3(blocks), t, 0, st, *a)));                             \
        return B2_OK;                                                                                                \
    }
    if (vec) {
        if (few) B2_ROWS(4, 1)
        B2_ROWS(4, 2)
        B2_ROWS(4, 4)
    } else {
        if (few) B2_ROWS(1, 2)
        B2_ROWS(1, 8)
        B2_ROWS(1, 16)
    }
#undef B2_ROWS
    B2_CUDA(b2::launch_after(norm_any_kernel, dim3(blocks), kThreads, 0, st, *a));
    return B2_OK;
}

extern "C" int b2_norm_bprop_scratch_bytes(const b2_norm* a, size_t* bytes) {
    B2_REQUIRE(bytes, "missing argument");
    B2_CHECK(check_norm(a));
    const GradPlan one = grad_plan(*a, 1), five = grad_plan(*a, 5);
    *bytes = (size_t)(one.ctas > five.ctas ? one.ctas : five.ctas) * 3 * a->features * sizeof(float) + 256;
    return B2_OK;
}

extern "C" int b2_norm_bprop(const b2_norm* a, const b2_norm_grads* d, void* scratch, size_t scratch_bytes, void* stream) {
    size_t need = 0;
    B2_CHECK(b2_norm_bprop_scratch_bytes(a, &need));
    B2_REQUIRE(d, "missing argument");
    B2_REQUIRE(scratch && scratch_bytes >= need, "the norm's gradient needs %zu bytes of scratch, got %zu", need, scratch_bytes);
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
    }
    B2_CHECK(b2::require_here(scratch, "the norm's scratch"));
    cudaStream_t st = (cudaStream_t)stream;
    float* sums = (float*)(((uintptr_t)scratch + 255) / 256 * 256);
    float* gate = a->gate_kind == B2_GATE_FEATURE ? d->d_gate : nullptr;
    const bool full = a->gate_kind == B2_GATE_FULL;
    const int tensors = (d->d_out ? 2 : 0) + (d->d_stream ? 1 : 0) + (a->block ? 1 : 0) + (full ? 1 : 0);
    const GradPlan p = grad_plan(*a, tensors);
    const float* x = a->block ? a->stream : a->residual;
    const int64_t x_stride = a->block ? a->stream_stride : a->residual_stride;
    const bool vec = a->features % 4 == 0 && rows_aligned(a->block, a->block_stride) && (!d->d_out || rows_aligned(x, x_stride)) &&
                     rows_aligned(d->d_out, d->d_out_stride) && rows_aligned(d->d_stream, d->d_stream_stride) &&
                     rows_aligned(d->d_residual, d->d_residual_stride) && rows_aligned(d->d_block, d->d_block_stride) &&
                     (full ? rows_aligned(a->gate, a->gate_stride) && rows_aligned(d->d_gate, d->d_gate_stride) : a->gate_kind == B2_GATE_ROW || b2::aligned16(a->gate)) &&
                     b2::aligned16(a->post_weight) && b2::aligned16(a->pre_weight);
    if (p.ctas > 0) {
        if (!p.threads) B2_CUDA(b2::launch_after(norm_grad_any_kernel, dim3(p.ctas), kThreads, 0, st, *a, *d, sums));
        else if (vec && p.each == 8) B2_CHECK((launch_grad<4, 2>(*a, *d, p, tensors, sums, st)));
        else if (vec) B2_CHECK((launch_grad<4, 4>(*a, *d, p, tensors, sums, st)));
        else if (p.each == 8) B2_CHECK((launch_grad<1, 8>(*a, *d, p, tensors, sums, st)));
        else B2_CHECK((launch_grad<1, 16>(*a, *d, p, tensors, sums, st)));
    }
    if (d->d_pre_weight || d->d_post_weight || gate)
        B2_CUDA(b2::launch_after(norm_sums_kernel, dim3((a->features + 31) / 32, 3), 1024, 0, st, (const float*)sums, p.ctas, a->features, d->d_pre_weight,
                                 d->d_post_weight, gate));
    return B2_OK;
}
