// The edge between two blocks of a residual network, and its gradients:
//
//   stream = a residual + gate * (rms(block) * w_post),   out = rms(stream) * w_pre,   rms(x) = x * rstd(x)
//
//   d_stream' = d_stream + through(d_out, stream, w_pre),  d_residual = a d_stream',  d_gate = d_stream' * rms(block) w_post
//   d_block   = through(gate * d_stream', block, w_post)
//   through(d, x, w) = rstd (w d - x^ mean(w d x^)),  x^ = x rstd;   d_w = sum over rows of d x^
#include <cstdint>

#include "b2_operators.h"

namespace {

constexpr int kThreads = 256;

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

__global__ void __launch_bounds__(kThreads)
norm_sums_kernel(const float* __restrict__ sums, int ctas, int F, float* pre, float* post, float* gate) {
    after_earlier_kernels();
    const int i = blockIdx.x * kThreads + threadIdx.x;
    if (i >= 3 * F) return;
    float s = 0.0f;
    for (int c = 0; c < ctas; ++c) s += sums[(long long)c * 3 * F + i];
    if (i < F) {
        if (pre) pre[i] = s;
    } else if (i < 2 * F) {
        if (post) post[i - F] = s;
    } else if (gate) {
        gate[i - 2 * F] = s;
    }
}

int ctas_of(const b2_norm& a) { return (int)(a.rows < b2::kSms * 4 ? a.rows : b2::kSms * 4); }

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
    const long long blocks = a->rows < (1ll << 30) ? a->rows : (1ll << 30);
    B2_CUDA(b2::launch_after(norm_any_kernel, dim3((unsigned)blocks), kThreads, 0, (cudaStream_t)stream, *a));
    return B2_OK;
}

extern "C" int b2_norm_bprop_scratch_bytes(const b2_norm* a, size_t* bytes) {
    B2_REQUIRE(bytes, "missing argument");
    B2_CHECK(check_norm(a));
    *bytes = (size_t)ctas_of(*a) * 3 * a->features * sizeof(float) + 256;
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
    const int ctas = ctas_of(*a);
    if (ctas > 0) B2_CUDA(b2::launch_after(norm_grad_any_kernel, dim3(ctas), kThreads, 0, st, *a, *d, sums));
    float* gate = a->gate_kind == B2_GATE_FEATURE ? d->d_gate : nullptr;
    if (d->d_pre_weight || d->d_post_weight || gate)
        B2_CUDA(b2::launch_after(norm_sums_kernel, dim3((3 * a->features + kThreads - 1) / kThreads), kThreads, 0, st, (const float*)sums, ctas, a->features,
                                 d->d_pre_weight, d->d_post_weight, gate));
    return B2_OK;
}
