// One AdamW step over many tensors.
//
//   m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2
//   p = p (1 - lr wd) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
//
// Bound by memory: 28 bytes a value with fp32 moments, 16.06 with moments in 8 bits.  The tensors are cut into chunks
// of 2048 values, one 64-byte record each, made once (the addresses of a program's tensors stay): a CTA reads a
// record and its values, whatever tensor they belong to, so that many small tensors cost no launches.  79.5 million values:
// 345 us with fp32 moments, 0.99 of the rate of a copy; 252 us with 8-bit ones, 0.78 of it (some 84 instructions a value, of
// which division and square root, correctly rounded, are a fifth, issued in 73 % of the cycles; in the others the warps wait
// for loads), and 284 where the power cap has lowered the clock to 1.7 GHz.  162 000 values: 3.7 us in a graph.
//
// Moments in 8 bits: a warp holds 256 values and their two scales.  m and sqrt(v) are e4m3 values times the block's
// largest / 448.  v itself spans the square of what its root does, and e4m3 covers 2.3e5 : 1.  An average with
// beta2 = 0.999 moves by at most 0.05 % of its root in a step downwards where e4m3's neighbours are 6 to 12 % apart: rounded to
// nearest it would never come down.  Rounded at random to either neighbour, with the chance that makes the mean
// right, it does, on the average.  That is the mean of m and of the root.  v is the root squared, and each rounding leaves
// its variance there: a value that moves by d against a grid of distance D is rounded with a variance of about d D, d some
// (1 - beta2) / 2 of the root and as much for the scale that the grid moves with, D 1/16 to 1/8 of it; over the 1 / (1 - beta2) steps that
// the average remembers, 4 to 6 % of v, 1 % of a step's size.  A root that is not zero is not rounded to zero, which would
// leave m / eps.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <new>
#include <vector>

#include <cuda_fp8.h>

#include "b2_operators.h"

namespace {

constexpr int kChunk = 2048;
constexpr int kThreads = 256;
constexpr int kBlock = 256;             // values with one scale

struct Chunk {
    float* param;
    const float* grad;
    void *m, *v;
    float *m_scales, *v_scales;
    unsigned n, counter;
    float decay;
    unsigned vec;                       // all addresses allow vectors
};
static_assert(sizeof(Chunk) == 64, "records are read as four vectors");
constexpr size_t kHeader = 256;         // of a plan: Header, then the records
struct Header {
    unsigned finished;                  // CTAs of the running step that have come to their end
    int state_bits;
    long long chunks;
};

struct Rates {
    float b1, c1, b2, c2, eps;
    double lr, wd, beta1, beta2;
};

struct Now {
    float size, root, lr_wd, grad_scale;
    unsigned key;
};

__device__ __forceinline__ unsigned mix(unsigned x) {
    x = (x ^ (x >> 16)) * 0x9E3779B9u;          // (odd words: multiplication permutes)
    x = (x ^ (x >> 15)) * 0xBB67AE85u;
    return x ^ (x >> 16);
}

// x^t by squaring
__device__ __forceinline__ double power(double x, unsigned t) {
    double y = 1.0;
    for (; t; t >>= 1, x *= x)
        if (t & 1) y *= x;
    return y;
}

// What depends on the number of the step, in 64 bits: 1 - beta^t cancels where beta^t is near 1.
__device__ __forceinline__ float begin_step(const Rates& r, const float* lr_at, const float* scale_at, const float* step, unsigned seed, Now* now) {
    const float before = *step;
    const unsigned t = before >= 0.0f ? (unsigned)fminf(before, 4.0e9f) + 1u : 1u;
    const double lr = lr_at ? (double)*lr_at : r.lr;
    now->size = (float)(lr / (1.0 - power(r.beta1, t)));
    now->root = (float)(1.0 / sqrt(1.0 - power(r.beta2, t)));
    now->lr_wd = (float)(lr * r.wd);
    now->grad_scale = scale_at ? *scale_at : 1.0f;
    const unsigned key = mix(seed + 0x9E3779B9u * t);
    now->key = key ^ (key >> 16);               // (as the first step of mix() leaves it)
    return before;
}

// The new moments, the root of the second, and the new value.  Every operation is rounded by itself: the result does
// not depend on how the values are spread over threads.
__device__ __forceinline__ float update(const Rates& r, const Now& now, float keep, float p, float g, float& m, float& v, float& root) {
    g = __fmul_rn(g, now.grad_scale);
    m = __fadd_rn(__fmul_rn(m, r.b1), __fmul_rn(g, r.c1));
    v = __fadd_rn(__fmul_rn(v, r.b2), __fmul_rn(__fmul_rn(g, g), r.c2));
    root = __fsqrt_rn(v);
    const float d = __fdiv_rn(m, __fadd_rn(__fmul_rn(root, now.root), r.eps));
    return __fsub_rn(__fmul_rn(p, keep), __fmul_rn(d, now.size));
}

// The step is counted by the CTA that finishes last: every other one has read the count by then.
__device__ __forceinline__ void end_step(Header* plan, int state_bits, float* step, float before) {
    if (threadIdx.x == 0 && atomicInc(&plan->finished, gridDim.x - 1) == gridDim.x - 1 && plan->state_bits == state_bits) *step = before + 1.0f;
}

// Records that a kernel may go through: those of the plan, however many the caller names; none of a plan for other moments.
__device__ __forceinline__ long long records(const Header* plan, long long named, int state_bits) {
    return plan->state_bits == state_bits ? min(named, plan->chunks) : 0;
}

__global__ void __launch_bounds__(kThreads)
adamw32_kernel(Header* plan, const Chunk* __restrict__ chunks, long long named, Rates r, const float* lr_at, const float* scale_at, float* step,
               unsigned seed) {
    __shared__ Now shared_now;
    after_earlier_kernels();
    float before = 0.0f;
    if (threadIdx.x == 0) before = begin_step(r, lr_at, scale_at, step, seed, &shared_now);
    __syncthreads();
    const Now now = shared_now;
    const long long n_chunks = records(plan, named, 32);
    for (long long k = blockIdx.x; k < n_chunks; k += gridDim.x) {
        const Chunk c = chunks[k];
        float* m = static_cast<float*>(c.m);
        float* v = static_cast<float*>(c.v);
        const float keep = __fsub_rn(1.0f, __fmul_rn(c.decay, now.lr_wd));
        float unused;
        if (c.vec) {
            constexpr int UN = kChunk / kThreads / 4;
            float4 p4[UN], g4[UN], m4[UN], v4[UN];
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const int i = (u * kThreads + threadIdx.x) * 4;
                if (i + 4 <= (int)c.n) {
                    p4[u] = *reinterpret_cast<const float4*>(c.param + i);
                    g4[u] = *reinterpret_cast<const float4*>(c.grad + i);
                    m4[u] = *reinterpret_cast<const float4*>(m + i);
                    v4[u] = *reinterpret_cast<const float4*>(v + i);
                }
            }
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const int i = (u * kThreads + threadIdx.x) * 4;
                if (i + 4 <= (int)c.n) {
                    p4[u].x = update(r, now, keep, p4[u].x, g4[u].x, m4[u].x, v4[u].x, unused);
                    p4[u].y = update(r, now, keep, p4[u].y, g4[u].y, m4[u].y, v4[u].y, unused);
                    p4[u].z = update(r, now, keep, p4[u].z, g4[u].z, m4[u].z, v4[u].z, unused);
                    p4[u].w = update(r, now, keep, p4[u].w, g4[u].w, m4[u].w, v4[u].w, unused);
                    *reinterpret_cast<float4*>(c.param + i) = p4[u];
                    *reinterpret_cast<float4*>(m + i) = m4[u];
                    *reinterpret_cast<float4*>(v + i) = v4[u];
                }
            }
        }
        for (int i = (c.vec ? (int)(c.n & ~3u) : 0) + threadIdx.x; i < (int)c.n; i += kThreads) {
            float mi = m[i], vi = v[i];
            c.param[i] = update(r, now, keep, c.param[i], c.grad[i], mi, vi, unused);
            m[i] = mi;
            v[i] = vi;
        }
    }
    end_step(plan, 32, step, before);
}

// The byte (without its sign) of one of the two neighbours in e4m3 of q, |q| <= 448 but for a rounding, in the uppermost byte:
// of the upper neighbour with the chance that sixteen random bits give it, here in the middle two bytes.  Times 2^-120,
// exponent and mantissa of an fp32 value have in bits 20 to 27 the byte of e4m3, fp32's denormals that of e4m3's, which
// are 2^-9 apart; what is below is added to and cut off.  (No carry beyond 448: the random bits end above the roundings
// of q.)
__device__ __forceinline__ unsigned to_e4m3(float q, unsigned bits) {
    return (__float_as_uint(__fmul_rn(fabsf(q), 7.52316384526264e-37f)) << 4) + bits;
}
// the uppermost bytes of four words
__device__ __forceinline__ unsigned tops(unsigned a, unsigned b, unsigned c, unsigned d) {
    return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
}

// Two products to an instruction.  Sums are taken one by one: the assembler joins a product and a sum of this form into one
// operation, rounded once, .rn or not (seen in the bits of v).
struct Two {
    unsigned long long w;
};
__device__ __forceinline__ Two two(float x, float y) {
    Two t;
    asm("mov.b64 %0, {%1, %2};" : "=l"(t.w) : "f"(x), "f"(y));
    return t;
}
__device__ __forceinline__ void apart(Two t, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(t.w)); }
__device__ __forceinline__ Two operator*(Two a, Two b) {
    Two t;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(t.w) : "l"(a.w), "l"(b.w));
    return t;
}
__device__ __forceinline__ Two operator+(Two a, Two b) {
    float a0, a1, b0, b1;
    apart(a, a0, a1);
    apart(b, b0, b1);
    return two(__fadd_rn(a0, b0), __fadd_rn(a1, b1));
}

// update() of two values
__device__ __forceinline__ Two update(const Rates& r, const Now& now, float keep, Two p, Two g, Two& m, Two& v, float& r0, float& r1) {
    auto both = [](float x) { return two(x, x); };
    g = g * both(now.grad_scale);
    m = m * both(r.b1) + g * both(r.c1);
    v = v * both(r.b2) + (g * g) * both(r.c2);
    float v0, v1, m0, m1, d0, d1;
    apart(v, v0, v1);
    apart(m, m0, m1);
    r0 = __fsqrt_rn(v0);
    r1 = __fsqrt_rn(v1);
    apart(two(r0, r1) * both(now.root) + both(r.eps), d0, d1);
    return p * both(keep) + two(__fdiv_rn(m0, d0), __fdiv_rn(m1, d1)) * both(-now.size);
}

// the larger magnitude, NaN where there is one
__device__ __forceinline__ float larger(float top, float x) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(x)));
    return top;
}

__device__ __forceinline__ float2 from_e4m3(unsigned two) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
    return __half22float2(__half2(h));
}
// What values are multiplied by, 448 (1 / top), and the scales, top (1 / 448), of both moments: one division, in different
// lanes for both.
__device__ __forceinline__ void scales_of(float top_m, float top_r, float& to_m, float& to_r, float& new_ms, float& new_vs) {
    const int lane = threadIdx.x & 31;
    const float top = lane & 1 ? top_r : top_m;
    const bool live = top > 7.888609052210118e-31f;             // 2^-100
    float x = live ? lane & 2 ? __fmul_rn(top, 1.0f / 448.0f) : __fmul_rn(__fdiv_rn(1.0f, top), 448.0f) : 0.0f;
    if ((lane & 2) && !(top <= 3.402823466e+38f)) x = __int_as_float(0x7fffffff);
    to_m = __shfl_sync(0xffffffffu, x, 0);
    to_r = __shfl_sync(0xffffffffu, x, 1);
    new_ms = __shfl_sync(0xffffffffu, x, 2);
    new_vs = __shfl_sync(0xffffffffu, x, 3);
}

__global__ void __launch_bounds__(kThreads, 4)
adamw8_kernel(Header* plan, const Chunk* __restrict__ chunks, long long named, Rates r, const float* lr_at, const float* scale_at, float* step,
              unsigned seed) {
    __shared__ Now shared_now;
    after_earlier_kernels();
    float before = 0.0f;
    if (threadIdx.x == 0) before = begin_step(r, lr_at, scale_at, step, seed, &shared_now);
    __syncthreads();
    const Now now = shared_now;
    const long long n_chunks = records(plan, named, 8);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (long long k = blockIdx.x; k < n_chunks; k += gridDim.x) {
        const Chunk c = chunks[k];
        const int at = warp * kBlock;
        // the next chunk's values on their way to the second cache, a line to a lane, and the record behind it to the first
        if (k + 2 * gridDim.x < n_chunks && lane == 31) asm volatile("prefetch.global.L1 [%0];" ::"l"(chunks + k + 2 * gridDim.x));
        if (k + gridDim.x < n_chunks && lane < 20) {
            const Chunk* next = chunks + k + gridDim.x;
            const int line = lane < 16 ? lane & 7 : lane & 1, from = at + line * (lane < 16 ? 32 : 128);
            const char* p = lane < 8 ? (const char*)(next->param + from) : lane < 16 ? (const char*)(next->grad + from)
                          : lane < 18 ? static_cast<const char*>(next->m) + from : static_cast<const char*>(next->v) + from;
            if (from < (int)next->n) asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
        }
        const int n = (int)c.n - at;                    // of the warp's block
        if (n <= 0) continue;
        unsigned char* mc = static_cast<unsigned char*>(c.m) + at;
        unsigned char* vc = static_cast<unsigned char*>(c.v) + at;
        const float keep = __fsub_rn(1.0f, __fmul_rn(c.decay, now.lr_wd));
        // a lane's values: four from 4 lane on, four from 128 + 4 lane on
        Two p[4], g[4], m[4], v[4];
        float root[8];
        const bool vec = c.vec && n >= kBlock;
        const float ms = c.m_scales[warp], vs = c.v_scales[warp];
        unsigned mw[2], vw[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = h * 128 + lane * 4;
            if (vec) {
                const float4 p4 = *reinterpret_cast<const float4*>(c.param + at + i), g4 = *reinterpret_cast<const float4*>(c.grad + at + i);
                p[2 * h] = two(p4.x, p4.y);
                p[2 * h + 1] = two(p4.z, p4.w);
                g[2 * h] = two(g4.x, g4.y);
                g[2 * h + 1] = two(g4.z, g4.w);
                mw[h] = *reinterpret_cast<const unsigned*>(mc + i);
                vw[h] = *reinterpret_cast<const unsigned*>(vc + i);
            } else {
                float x[4], y[4];
                mw[h] = vw[h] = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bool there = i + j < n;
                    x[j] = there ? c.param[at + i + j] : 0.0f;
                    y[j] = there ? c.grad[at + i + j] : 0.0f;
                    mw[h] |= there ? (unsigned)mc[i + j] << (8 * j) : 0u;
                    vw[h] |= there ? (unsigned)vc[i + j] << (8 * j) : 0u;
                }
                p[2 * h] = two(x[0], x[1]);
                p[2 * h + 1] = two(x[2], x[3]);
                g[2 * h] = two(y[0], y[1]);
                g[2 * h + 1] = two(y[2], y[3]);
            }
        }
        float most_m = 0.0f, most_r = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 mf = from_e4m3(mw[e / 2] >> (16 * (e & 1)) & 0xffff), rf = from_e4m3(vw[e / 2] >> (16 * (e & 1)) & 0xffff);
            m[e] = two(mf.x, mf.y) * two(ms, ms);
            const Two old = two(rf.x, rf.y) * two(vs, vs);
            v[e] = old * old;
            p[e] = update(r, now, keep, p[e], g[e], m[e], v[e], root[2 * e], root[2 * e + 1]);
            float m0, m1;
            apart(m[e], m0, m1);
            most_m = larger(larger(most_m, m0), m1);
            most_r = larger(larger(most_r, root[2 * e]), root[2 * e + 1]);
        }
        // as bits, whose order is that of the values (NaN above all)
        const unsigned top_m = __reduce_max_sync(0xffffffffu, __float_as_uint(most_m)), top_r = __reduce_max_sync(0xffffffffu, __float_as_uint(most_r));
        float to_m, to_r, new_ms, new_vs;
        scales_of(__uint_as_float(top_m), __uint_as_float(top_r), to_m, to_r, new_ms, new_vs);
        if (lane == 0) {
            c.m_scales[warp] = new_ms;
            c.v_scales[warp] = new_vs;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = h * 128 + lane * 4;
            unsigned mb[4], vb[4], qm_bits[4];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float qm[2], qr[2];
                apart(m[2 * h + k] * two(to_m, to_m), qm[0], qm[1]);
                apart(two(root[4 * h + 2 * k], root[4 * h + 2 * k + 1]) * two(to_r, to_r), qr[0], qr[1]);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    // mix() of position and key, the first and the last of its steps put together with what is next to them:
                    // its upper half rounds the root, its lower half the average
                    const unsigned at_e = c.counter + (unsigned)(at + i + 2 * k + j);
                    unsigned y = (at_e ^ (at_e >> 16) ^ now.key) * 0x9E3779B9u;
                    y = (y ^ (y >> 15)) * 0xBB67AE85u;
                    qm_bits[2 * k + j] = __float_as_uint(qm[j]);
                    mb[2 * k + j] = to_e4m3(qm[j], __byte_perm(y ^ (y >> 16), 0u, 0x4104));
                    vb[2 * k + j] = max(to_e4m3(qr[j], __byte_perm(y, 0u, 0x4324)), min(__float_as_uint(qr[j]), 1u) << 24);
                }
            }
            const unsigned mo = (tops(mb[0], mb[1], mb[2], mb[3]) & 0x7f7f7f7fu) |
                                (tops(qm_bits[0], qm_bits[1], qm_bits[2], qm_bits[3]) & 0x80808080u);
            const unsigned vo = tops(vb[0], vb[1], vb[2], vb[3]);
            float x[4];
            apart(p[2 * h], x[0], x[1]);
            apart(p[2 * h + 1], x[2], x[3]);
            if (vec) {
                *reinterpret_cast<float4*>(c.param + at + i) = make_float4(x[0], x[1], x[2], x[3]);
                *reinterpret_cast<unsigned*>(mc + i) = mo;
                *reinterpret_cast<unsigned*>(vc + i) = vo;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (i + j < n) {
                        c.param[at + i + j] = x[j];
                        mc[i + j] = (unsigned char)(mo >> (8 * j));
                        vc[i + j] = (unsigned char)(vo >> (8 * j));
                    }
            }
        }
    }
    end_step(plan, 8, step, before);
}

int count_chunks(const b2_adamw_tensor* list, int count, int state_bits, long long* chunks) {
    B2_REQUIRE(count >= 0 && (count == 0 || list), "bad list of tensors");
    B2_REQUIRE(state_bits == 32 || state_bits == 8, "moments are held in 32 or 8 bits, not in %d", state_bits);
    *chunks = 0;
    for (int i = 0; i < count; ++i) {
        const b2_adamw_tensor& t = list[i];
        B2_REQUIRE(t.n >= 0, "tensor %d has %lld values", i, (long long)t.n);
        B2_REQUIRE(t.n == 0 || (t.param && t.grad && t.m && t.v), "tensor %d: missing address", i);
        B2_REQUIRE(t.n == 0 || state_bits == 32 || (t.m_scales && t.v_scales), "tensor %d: missing scales", i);
        *chunks += (t.n + kChunk - 1) / kChunk;
    }
    return B2_OK;
}

}  // namespace

// Blocks write in any order: what one writes no other may read or write.  The plan holds addresses that are written to.
static int check_apart(const b2_adamw_tensor* tensors, int32_t count, int32_t state_bits, const void* plan, size_t plan_bytes) {
    struct Range {
        uintptr_t from, to;
        bool operator<(const Range& o) const { return from < o.from; }
    };
    const auto range = [](const void* p, size_t bytes) { return Range{(uintptr_t)p, (uintptr_t)p + bytes}; };
    std::vector<Range> written = {range(plan, plan_bytes)};
    for (int i = 0; i < count; ++i) {
        const b2_adamw_tensor& t = tensors[i];
        if (t.n == 0) continue;
        const size_t values = (size_t)t.n, scales = (values + kBlock - 1) / kBlock * 4, moments = state_bits == 32 ? 4 * values : values;
        written.push_back(range(t.param, 4 * values));
        written.push_back(range(t.m, moments));
        written.push_back(range(t.v, moments));
        if (state_bits == 8) {
            written.push_back(range(t.m_scales, scales));
            written.push_back(range(t.v_scales, scales));
        }
    }
    std::sort(written.begin(), written.end());
    for (size_t k = 1; k < written.size(); ++k)
        B2_REQUIRE(written[k - 1].to <= written[k].from, "tensors of the plan overlap, or lie in its memory");
    for (int i = 0; i < count; ++i) {
        if (tensors[i].n == 0) continue;
        const Range g = range(tensors[i].grad, 4 * (size_t)tensors[i].n);
        const auto next = std::lower_bound(written.begin(), written.end(), Range{g.to, 0});     // the first that begins behind it
        B2_REQUIRE(next == written.begin() || (next - 1)->to <= g.from, "gradient %d overlaps a tensor that the step writes", i);
    }
    return B2_OK;
}

// Addresses between two values would fault on the device.
static bool whole(const void* p, size_t bytes) { return (uintptr_t)p % bytes == 0; }

extern "C" int b2_adamw_plan_bytes(const b2_adamw_tensor* tensors, int32_t count, int32_t state_bits, size_t* bytes, int64_t* chunks) {
    B2_REQUIRE(bytes && chunks, "bad argument");
    long long n = 0;
    B2_CHECK(count_chunks(tensors, count, state_bits, &n));
    *chunks = n;
    *bytes = kHeader + (size_t)n * sizeof(Chunk) + 64;
    return B2_OK;
}

static char* plan_base(void* plan) { return (char*)(((uintptr_t)plan + 63) / 64 * 64); }

extern "C" int b2_adamw_plan(const b2_adamw_tensor* tensors, int32_t count, int32_t state_bits, void* plan, size_t plan_bytes, void* stream) {
    size_t need = 0;
    int64_t chunks = 0;
    B2_CHECK(b2_adamw_plan_bytes(tensors, count, state_bits, &need, &chunks));
    B2_REQUIRE(plan && plan_bytes >= need, "the plan needs %zu bytes, got %zu", need, plan_bytes);
    try {
        B2_CHECK(check_apart(tensors, count, state_bits, plan, need));
    } catch (const std::bad_alloc&) {
        return b2::fail(B2_ERR_INVALID, "no memory for a plan of %d tensors", count);
    }
    for (int i = 0; i < count; ++i) {
        const b2_adamw_tensor& t = tensors[i];
        if (t.n == 0) continue;
        const bool states = state_bits == 32 ? whole(t.m, 4) && whole(t.v, 4) : whole(t.m_scales, 4) && whole(t.v_scales, 4);
        B2_REQUIRE(whole(t.param, 4) && whole(t.grad, 4) && states, "tensor %d lies between two addresses", i);
    }
    b2::Memory memory;
    B2_CHECK(memory.find_device());
    B2_CHECK(memory.written(plan, "the plan"));
    for (int i = 0; i < count; ++i) {
        if (tensors[i].n == 0) continue;
        B2_CHECK(memory.written(tensors[i].param, "a tensor of the plan"));
        B2_CHECK(memory.read(tensors[i].grad, "a gradient of the plan"));
        B2_CHECK(memory.written(tensors[i].m, "a moment of the plan"));
        B2_CHECK(memory.written(tensors[i].v, "a moment of the plan"));
        if (state_bits == 8) {
            B2_CHECK(memory.written(tensors[i].m_scales, "the scales of a moment"));
            B2_CHECK(memory.written(tensors[i].v_scales, "the scales of a moment"));
        }
    }
    cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
    B2_CUDA(cudaStreamIsCapturing((cudaStream_t)stream, &capturing));
    B2_REQUIRE(capturing == cudaStreamCaptureStatusNone, "a plan is made before its stream is captured");
    try {
        std::vector<char> host(kHeader + (size_t)chunks * sizeof(Chunk), 0);
        *reinterpret_cast<Header*>(host.data()) = {0, state_bits, (long long)chunks};
        Chunk* c = reinterpret_cast<Chunk*>(host.data() + kHeader);
        for (int i = 0; i < count; ++i) {
            const b2_adamw_tensor& t = tensors[i];
            for (int64_t at = 0; at < t.n; at += kChunk, ++c) {
                const size_t state = state_bits == 32 ? 4 : 1;
                c->param = t.param + at;
                c->grad = t.grad + at;
                c->m = static_cast<char*>(t.m) + at * state;
                c->v = static_cast<char*>(t.v) + at * state;
                if (state_bits == 8) {
                    c->m_scales = t.m_scales + at / kBlock;
                    c->v_scales = t.v_scales + at / kBlock;
                }
                c->n = (unsigned)(t.n - at < kChunk ? t.n - at : kChunk);
                c->counter = t.counter + (unsigned)at;
                c->decay = t.decay;
                const uintptr_t states = (uintptr_t)c->m | (uintptr_t)c->v;
                c->vec = b2::aligned16(c->param) && b2::aligned16(c->grad) && states % (4 * state) == 0;
            }
        }
        // (pageable memory: the copy has been staged when the call returns)
        B2_CUDA(cudaMemcpyAsync(plan_base(plan), host.data(), host.size(), cudaMemcpyHostToDevice, (cudaStream_t)stream));
        B2_CUDA(cudaStreamSynchronize((cudaStream_t)stream));
    } catch (const std::bad_alloc&) {
        return b2::fail(B2_ERR_INVALID, "no memory for a plan of %zu bytes", need);
    }
    return B2_OK;
}

extern "C" int b2_adamw_step(void* plan, int64_t chunks, int32_t state_bits, const b2_adamw_hyper* h, const float* lr, const float* grad_scale, float* step,
                             uint32_t seed, void* stream) {
    B2_REQUIRE(plan && h && step && chunks >= 0, "bad argument");
    B2_REQUIRE(state_bits == 32 || state_bits == 8, "moments are held in 32 or 8 bits, not in %d", state_bits);
    B2_REQUIRE(h->beta1 >= 0.0 && h->beta1 < 1.0 && h->beta2 >= 0.0 && h->beta2 < 1.0 && h->eps >= 0.0 && std::isfinite(h->lr) &&
                   std::isfinite(h->weight_decay) && std::isfinite(h->eps),
               "bad rates: lr %g, beta1 %g, beta2 %g, eps %g, weight decay %g", h->lr, h->beta1, h->beta2, h->eps, h->weight_decay);
    B2_REQUIRE(whole(step, 4) && whole(lr, 4) && whole(grad_scale, 4), "a number of the step lies between two addresses");
    b2::Memory memory;
    B2_CHECK(memory.find_device());
    B2_CHECK(memory.written(step, "the number of the step"));
    B2_CHECK(memory.written(plan, "the plan"));
    B2_CHECK(memory.read(lr, "the rate"));
    B2_CHECK(memory.read(grad_scale, "the scale of the gradients"));
    Rates r;
    r.b1 = (float)h->beta1;
    r.c1 = (float)(1.0 - h->beta1);
    r.b2 = (float)h->beta2;
    r.c2 = (float)(1.0 - h->beta2);
    r.eps = (float)h->eps;
    r.lr = h->lr;
    r.wd = h->weight_decay;
    r.beta1 = h->beta1;
    r.beta2 = h->beta2;
    char* base = plan_base(plan);
    long long blocks = chunks < 1 ? 1 : chunks;
    if (blocks > b2::kSms * 8) blocks = b2::kSms * 8;
    B2_CUDA(b2::launch_after(state_bits == 32 ? adamw32_kernel : adamw8_kernel, dim3((unsigned)blocks), kThreads, 0, (cudaStream_t)stream,
                             reinterpret_cast<Header*>(base), reinterpret_cast<const Chunk*>(base + kHeader), (long long)chunks, r, lr, grad_scale, step, seed));
    return B2_OK;
}
