// Rotation of heads by position, and the norm of every head with the rotation in the same pass:
//
//   rotary     z_i -> amplitude z_i exp(i angle),  angle = position * frequency_i,  z_i a pair of features
//   forward    y = rotated(x^ w),  x^ = x rstd,  rstd = 1 / sqrt(mean(x^2) + eps)
//   gradients  d = rotated back(dy),  dw = sum over rows and heads of d x^,  dx = rstd (w d - x^ mean(w d x^))
//
// Angles: a frequency is a 64-bit fraction of a turn, so that the product with a position, modulo 2^64, is the fraction of a
// turn that is left, exact but for the frequency, which is good to 2^-61 of a turn (2^-41 at position a million).  In fp32
// position * frequency would be 0.03 radians off there.  The nearest quarter turn is taken off as an integer and the rest,
// at most an eighth of a turn, goes into the series of sine and cosine.
//
// Bound by memory: 8 bytes a value forward, 12 backward, each tensor read once and its angles worked out from 8 bytes a row.  8192
// rows, heads of 128: rotation of 16 + 4 heads 28.9 us (168 MB, 5.8 TB/s), norm and rotation of 32 + 8 59.8 (337 MB, 5.6), their
// gradients 105 (505 MB, 4.8), where a copy has 6.55.  A lane takes the same features of several heads, so that the angles, some
// twenty instructions a pair, are shared by the heads of a row; what is left between this and a copy is instructions (each of four
// schedulers issues in about half of its cycles, with 8 to 16 warps) and, of gradients, the sums over CTAs in a second launch.
#include <cmath>
#include <cstdint>
#include <limits>
#include <type_traits>

#include "b2_operators.h"
#include "b2_ew_device.cuh"

namespace {

using b2::Rows;
using b2::rows_at;
using b2::check_apart;

constexpr int kMostDim = 1024;
constexpr int kWarps = 4;           // of a CTA of the kernel for heads of any length

struct FlexArgs {
    const b2_flex_scale* table;
    int* stats;
    unsigned long long* probe_out;
    int probe;
};

// Which position a row has; false: none that 64 bits hold.
__device__ __forceinline__ bool position_of(const b2_heads& a, long long row, const b2_flex_scale* scales, long long& at) {
    unsigned long long i = (unsigned long long)row;
    if (a.position_group != 1) i /= (unsigned long long)a.position_group;
    if (i >= (unsigned long long)a.position_count) i %= (unsigned long long)a.position_count;
    at = (long long)i;
    if (!a.positions) return true;
    switch (a.position_kind) {
        case B2_IDX_I32: at = static_cast<const int*>(a.positions)[i]; return true;
        case B2_IDX_I64: at = static_cast<const long long*>(a.positions)[i]; return true;
        default: {
            const float x = a.position_kind == B2_IDX_F32 ? static_cast<const float*>(a.positions)[i]
                                                          : scales[a.slot_positions].scale * (float)static_cast<const short*>(a.positions)[i];
            at = __float2ll_rn(x);
            return x >= -0x1p63f && x < 0x1p63f;        // (false for NaN)
        }
    }
}

// amplitude * (cos, sin) of the fraction of a turn whose 64 bits are `phase`: of what is left of the nearest quarter turn by
// their series, up to x^9 / 9! and x^10 / 10!, whose next terms are 2e-9 and 5e-10 at an eighth of a turn.  (sincospif would look for
// the quarter turn again: the forward pass of 8192 x 40 heads of 128 takes 60.6 us with it, 59.9 so.)
__device__ __forceinline__ float2 turn_of(unsigned long long phase, float amplitude) {
    const unsigned t = (unsigned)(phase >> 32);
    const unsigned quarter = (t + 0x20000000u) >> 30;                                     // 0 ... 3: the fourth is the first
    const float x = (float)(int)(t - (quarter << 30)) * 1.4629180792671596e-9f;           // 2 pi / 2^32
    const float z = x * x;
    float s = fmaf(z, 2.7557319e-6f, -1.9841270e-4f), c = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
    s = fmaf(z, s, 8.3333333e-3f);
    c = fmaf(z, c, -1.3888889e-3f);
    s = fmaf(z, s, -1.6666667e-1f);
    c = fmaf(z, c, 4.1666667e-2f);
    s = fmaf(x * z, s, x);
    c = fmaf(z, c, -0.5f);
    c = fmaf(z, c, 1.0f);
    const bool swap = quarter & 1;
    const float u = swap ? s : c, v = swap ? c : s;
    return make_float2(amplitude * ((quarter + 1) & 2 ? -u : u), amplitude * (quarter & 2 ? -v : v));
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// fp32 to a mantissa, to the nearest even one; `stat` follows the largest
template <typename T> __device__ __forceinline__ T held(float v, float& stat);
template <> __device__ __forceinline__ float held<float>(float v, float&) { return v; }
template <> __device__ __forceinline__ short held<short>(float v, float& stat) { return (short)b2_f32_to_i16(v, stat); }

enum { ROTATE = 0, FORWARD = 1, BACKWARD = 2 };

// Heads of any length and alignment: a warp to a head, a lane to the pairs (lane, lane + 32, ...), and to what is not
// rotated; the sums of a norm read the head a second time.  The angles of a row are worked out once, by its CTA.
template <int MODE, typename T>
__global__ void __launch_bounds__(kWarps * 32)
heads_any_kernel(const b2_heads a, const b2_heads_grads g, const FlexArgs flex, float* __restrict__ sums) {
    extern __shared__ float2 table[];           // (cos, sin) of the row's pairs; BACKWARD: sums of a warp behind them
    after_earlier_kernels();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int D = a.head_dim, pairs = a.rotary_dim / 2, heads = a.part[0].heads + (a.parts > 1 ? a.part[1].heads : 0);
    float* mine = reinterpret_cast<float*>(table + pairs) + warp * 2 * D;
    if constexpr (MODE == BACKWARD) {
        for (int i = lane; i < 2 * D; i += 32) mine[i] = 0.0f;
        __syncwarp();
    }
    float factor = 1.0f, stat = 0.0f;
    if constexpr (sizeof(T) == 2) factor = flex.table[a.part[0].slot_x].scale * (flex.probe ? 1.0f : flex.table[a.part[0].slot_out].inv_scale);
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        if (pairs) {
            __syncthreads();                    // (the row before has been read)
            long long at;
            const bool good = position_of(a, row, flex.table, at);
            for (int i = threadIdx.x; i < pairs; i += kWarps * 32) {
                float2 w = turn_of((unsigned long long)at * a.turns[i], a.amplitude);
                if (MODE == BACKWARD || a.inverse) w.y = -w.y;
                table[i] = good ? w : make_float2(NAN, NAN);
            }
            __syncthreads();
        }
        for (int head = blockIdx.y * kWarps + warp; head < heads; head += gridDim.y * kWarps) {
            const int n = head >= a.part[0].heads;
            const b2_heads_part& p = a.part[n];
            const int h = head - (n ? a.part[0].heads : 0);
            const T* x = static_cast<const T*>(p.x) + row * p.x_row + h * p.x_head;
            const T* in = x;
            T* out = static_cast<T*>(p.out) + row * p.out_row + h * p.out_head;
            float rstd = 1.0f, mean = 0.0f;
            if constexpr (MODE == FORWARD) {
                float q = 0.0f;
                for (int i = lane; i < D; i += 32) q = fmaf((float)x[i], (float)x[i], q);
                rstd = __frsqrt_rn(__fdividef(warp_sum(q), (float)D) + a.eps);
                if (p.rstd && lane == 0) p.rstd[row * p.heads + h] = rstd;
            }
            if constexpr (MODE == BACKWARD) {
                rstd = p.rstd[row * p.heads + h];
                in = reinterpret_cast<const T*>(g.part[n].d_out) + row * g.part[n].d_out_row + h * g.part[n].d_out_head;
                out = g.part[n].d_x ? reinterpret_cast<T*>(g.part[n].d_x) + row * g.part[n].d_x_row + h * g.part[n].d_x_head : nullptr;
            }
            // (the rotation mixes two features of one lane)
            auto places = [&](auto&& visit) {
                for (int i = lane; i < pairs; i += 32) {
                    const int e = a.interleaved ? 2 * i : i;
                    visit(e, a.interleaved ? e + 1 : e + pairs, table[i]);
                }
                for (int i = 2 * pairs + lane; i < D; i += 32) visit(i, -1, make_float2(1.0f, 0.0f));
            };
            if constexpr (MODE == BACKWARD) {
                float q = 0.0f;
                places([&](int e, int f, float2 w) {
                    const float u = (float)in[e], v = f >= 0 ? (float)in[f] : 0.0f;
                    const float d = fmaf(u, w.x, -v * w.y), xe = (float)x[e] * rstd;
                    q = fmaf(p.weight ? p.weight[e] * d : d, xe, q);
                    mine[n * D + e] = fmaf(d, xe, mine[n * D + e]);
                    if (f >= 0) {
                        const float d2 = fmaf(v, w.x, u * w.y), xf = (float)x[f] * rstd;
                        q = fmaf(p.weight ? p.weight[f] * d2 : d2, xf, q);
                        mine[n * D + f] = fmaf(d2, xf, mine[n * D + f]);
                    }
                });
                mean = __fdividef(warp_sum(q), (float)D);
                if (!out) continue;
            }
            places([&](int e, int f, float2 w) {
                float u = (float)in[e], v = f >= 0 ? (float)in[f] : 0.0f;
                if constexpr (MODE == FORWARD) {
                    u *= p.weight ? rstd * p.weight[e] : rstd;
                    if (f >= 0) v *= p.weight ? rstd * p.weight[f] : rstd;
                }
                float y = f >= 0 ? fmaf(u, w.x, -v * w.y) : u, z = fmaf(v, w.x, u * w.y);
                if constexpr (MODE == BACKWARD) {
                    y = rstd * ((p.weight ? p.weight[e] * y : y) - (float)x[e] * rstd * mean);
                    if (f >= 0) z = rstd * ((p.weight ? p.weight[f] * z : z) - (float)x[f] * rstd * mean);
                }
                if constexpr (sizeof(T) == 2) {
                    y *= factor;
                    z = f >= 0 ? z * factor : 0.0f;
                    if (flex.probe) {
                        stat = fmaxf(stat, fmaxf(fabsf(y), fabsf(z)));
                        return;
                    }
                }
                out[e] = held<T>(y, stat);
                if (f >= 0) out[f] = held<T>(z, stat);
            });
        }
    }
    if constexpr (MODE == BACKWARD) {
        __syncthreads();
        const float* first = reinterpret_cast<const float*>(table + pairs);
        float* to = sums + (long long)(blockIdx.y * gridDim.x + blockIdx.x) * 2 * D;
        for (int i = threadIdx.x; i < 2 * D; i += kWarps * 32) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) v += first[w * 2 * D + i];
            to[i] = v;
        }
    }
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) stat = fmaxf(stat, __shfl_xor_sync(0xffffffffu, stat, o));
        if (lane == 0 && stat > 0.0f) {
            if (flex.probe) atomicMax(flex.probe_out, (unsigned long long)__float_as_uint(stat));
            else atomicMax(flex.stats + a.part[0].slot_out, (int)rintf(stat));
        }
    }
}

// How a launch deals out heads: `lanes` (as a power of two) to a head, so that a warp takes 32 >> lanes heads of one tensor at a
// time, `turns` times: that is a task.  Tasks are of one row, or, where a row's heads would leave many lanes without one, of heads next
// to one another whatever their rows (FLAT).
struct Deal {
    int lanes, turns;
    int ahead;                                      // whether the next task's heads are fetched into L2
    int narrow;                                     // 32 bits number what is divided
    long long first_tasks, row_tasks;               // of the first tensor (in a row, or FLAT in all), of a row
    long long tasks;
};
constexpr int kThreads = 256;
// Heads that a lane loads at once, by how many features of each it holds, and CTAs to an SM.  Eight features, 8192 rows of 40 heads of
// 128 forward, four heads: 59.9 us with two CTAs, 63.0 with three; two heads and four CTAs 78; one and five 108.  Gradients,
// two heads and two CTAs, for which shared memory has room: 105; one and three 144.  Rotation alone, 8192 x 20, four heads: 28.9 with
// three CTAs, 29.1 with two.
__host__ __device__ constexpr int unrolled(int mode, int values) { return mode == BACKWARD && values >= 8 ? 2 : 4; }
__host__ __device__ constexpr int blocks_to(int mode, int values) { return values < 8 ? (mode == BACKWARD ? 2 : 3) : mode == ROTATE ? 3 : 2; }
// How many tasks' heads a warp of whole vectors of a row has in shared memory or on their way there, of gradients: x, d_out and rstd
constexpr int kAhead = 3;
__host__ __device__ constexpr bool runs_ahead(int mode, int vec, bool flat) { return mode == BACKWARD && vec == 4 && !flat; }
constexpr int kSlotBytes = (2 * 32 * 16 * 2 + 32 * 4) * unrolled(BACKWARD, 8);
// CTAs that stay, and fetch the heads of their next task into L2 meanwhile: forward 65.8 us without, 59.9 with; a rotation, which waits
// for nothing but its loads, 28.9 without and 32.4 with.  (Of gradients a sum a CTA is stored, so that there are few of them.)
__host__ __device__ constexpr bool stays(int mode) { return mode != ROTATE; }

template <int VEC, typename T>
__device__ __forceinline__ void get(const T* p, float* v) {
    if constexpr (VEC == 1) {
        v[0] = (float)*p;
    } else if constexpr (sizeof(T) == 4) {
        const float4 w = *reinterpret_cast<const float4*>(p);
        v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
    } else {
        const int2 w = *reinterpret_cast<const int2*>(p);
        v[0] = (float)(short)(w.x & 0xffff);
        v[1] = (float)(w.x >> 16);
        v[2] = (float)(short)(w.y & 0xffff);
        v[3] = (float)(w.y >> 16);
    }
}
template <int VEC, typename T>
__device__ __forceinline__ void put(T* p, const float* v, float& stat) {
    if constexpr (VEC == 1) {
        *p = held<T>(v[0], stat);
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
        short q[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) q[k] = held<T>(v[k], stat);
        *reinterpret_cast<short4*>(p) = make_short4(q[0], q[1], q[2], q[3]);
    }
}

// Two values next to one another, for instructions that take two at a time
__device__ __forceinline__ float2 two(const float* v) { return make_float2(v[0], v[1]); }
__device__ __forceinline__ void apart(float2 w, float* v) { v[0] = w.x; v[1] = w.y; }

// Heads of up to 256 features: a lane holds the same features of every head that it comes to, EACH times two runs of VEC features
// that hold both features of their pairs, so that it works out its angles once a task, while the loads are on their way, and neither
// shares them nor waits for anybody.  All loads of a task are issued before the first is needed.
//   HALVES: a run lies as far from the other as the features of a pair; the features behind the rotated ones likewise
//   else:   VEC 4: two runs half a head apart, each of two pairs; VEC 1: a pair
// BACKWARD: sums for the weights stay in registers and are added over the CTA at the end.
template <int MODE, typename T, int VEC, int EACH, bool HALVES, bool FLAT>
__global__ void __launch_bounds__(kThreads, blocks_to(MODE, 2 * VEC * EACH))
heads_kernel(const b2_heads a, const b2_heads_grads g, const FlexArgs flex, const Deal deal, float* __restrict__ sums) {
    constexpr int N = 2 * VEC * EACH, P = N / 2, U = unrolled(MODE, N);
    static_assert(VEC == 1 || EACH == 1, "one pair of vectors");
    constexpr bool APART = VEC == 4 && HALVES;                  // the features of pair k: k and VEC + k, else 2 k and 2 k + 1
    after_earlier_kernels();
    const int lane = threadIdx.x & 31, sub = lane & ((1 << deal.lanes) - 1), beside = 32 >> deal.lanes, mine = lane >> deal.lanes;
    const int D = a.head_dim, r = a.rotary_dim;
    // where this lane's runs of features begin (-1: none), and its pairs' frequencies
    int at[2 * EACH];
    unsigned long long frequency[P];
    unsigned turning = 0;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int i = VEC * (sub + 32 * e);                     // of the first run
        int first, second;
        if (HALVES) {
            const int rest = (D - r + 1) / 2, j = i - r / 2;
            first = i < r / 2 ? i : j < rest ? r + j : -1;
            second = i < r / 2 ? i + r / 2 : j < rest && r + rest + j < D ? r + rest + j : -1;
        } else if (VEC == 4) {
            first = i < D / 2 ? i : -1;
            second = i < D / 2 ? D / 2 + i : -1;
        } else {
            first = 2 * i < D ? 2 * i : -1;
            second = 2 * i + 1 < D ? 2 * i + 1 : -1;
        }
        at[2 * e] = first;
        at[2 * e + 1] = second;
#pragma unroll
        for (int k = 0; k < P / EACH; ++k) {
            const int feature = HALVES ? first + k : VEC == 4 ? (k < 2 ? first + 2 * k : second + 2 * k - 4) : first;
            const bool turns = first >= 0 && feature < (HALVES ? r / 2 : r);
            frequency[e * (P / EACH) + k] = turns ? a.turns[HALVES ? feature : feature / 2] : 0;
            turning |= (unsigned)turns << (e * (P / EACH) + k);
        }
    }
    float acc[2][MODE == BACKWARD ? N : 1];
#pragma unroll
    for (int j = 0; j < (MODE == BACKWARD ? N : 1); ++j) acc[0][j] = acc[1][j] = 0.0f;
    float factor = 1.0f, stat = 0.0f;
    if constexpr (sizeof(T) == 2) factor = flex.table[a.part[0].slot_x].scale * (flex.probe ? 1.0f : flex.table[a.part[0].slot_out].inv_scale);

    const auto load = [&](const T* from, float* v) {
#pragma unroll
        for (int e = 0; e < 2 * EACH; ++e)
            if (at[e] >= 0) get<VEC>(from + at[e], v + VEC * e);
            else
#pragma unroll
                for (int k = 0; k < VEC; ++k) v[VEC * e + k] = 0.0f;
    };
    const float share = 1.0f / (float)D;
    // A warp's tasks: every so manieth; where they come by way of shared memory, so many next to one another, whose rows and angles are
    // often the same (3 us of 105; the forward pass takes as long either way, 59.9 and 60.1)
    constexpr bool RING = runs_ahead(MODE, VEC, FLAT);
    const long long warps = (long long)gridDim.x * (kThreads / 32), run = (deal.tasks + warps - 1) / warps, me = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    const long long task0 = RING ? me * run : me, end = RING && task0 + run < deal.tasks ? task0 + run : deal.tasks, step = RING ? 1 : warps;
    const int each = deal.turns * beside;                   // heads of a task
    const auto quotient = [&](long long i, long long by) { return deal.narrow ? (long long)((unsigned)i / (unsigned)by) : i / by; };
    // The tensor of a task, its row, and of its first head the place in the row or, FLAT, in the tensor
    struct Begin {
        int n;
        long long row;
        typename std::conditional<FLAT, long long, int>::type head;
    };
    const auto begin_of = [&](long long task) {
        Begin t;
        t.row = FLAT ? 0 : quotient(task, deal.row_tasks);
        if constexpr (FLAT) {
            t.n = task >= deal.first_tasks;
            t.head = (task - (t.n ? deal.first_tasks : 0)) * each;
        } else {
            const int in = (int)(task - t.row * deal.row_tasks), first_tasks = (int)deal.first_tasks;
            t.n = in >= first_tasks;
            t.head = (in - (t.n ? first_tasks : 0)) * each;
        }
        return t;
    };
    // Whole vectors of a row's heads come by way of shared memory, kAhead - 1 tasks ahead: a lane copies what it will read itself, so that
    // it waits for nobody else.
    extern __shared__ float2 table[];
    char* slots = reinterpret_cast<char*>(table) + (threadIdx.x >> 5) * (RING ? kAhead * kSlotBytes : 0) + lane * 16;
    const auto slot_of = [&](int stage, int tensor, int u, int e) { return slots + stage * kSlotBytes + ((tensor * U + u) * 2 + e) * 512; };
    const auto rstd_slot = [&](int stage, int u) { return slots + stage * kSlotBytes + 2 * U * 2 * 512 + u * 128 - lane * 12; };
    const auto copy_ahead = [&](long long task, int stage) {
        if (task < end) {
            const Begin t = begin_of(task);
            const b2_heads_part& p = a.part[t.n];
            const b2_heads_part_grads& d = g.part[t.n];
            const int first = (int)t.head + mine, left = p.heads - first;
            const auto copy = [&](const T* from, int tensor, long long head_stride) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const bool live = u < deal.turns && u * beside < left;
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((unsigned)__cvta_generic_to_shared(slot_of(stage, tensor, u, e))),
                                     "l"(live && at[e] >= 0 ? from + u * beside * head_stride + at[e] : static_cast<const T*>(p.x)), "r"(live && at[e] >= 0 ? 16 : 0)
                                     : "memory");
                }
            };
            copy(static_cast<const T*>(p.x) + t.row * p.x_row + first * p.x_head, 0, p.x_head);
            copy(reinterpret_cast<const T*>(d.d_out) + t.row * d.d_out_row + first * d.d_out_head, 1, d.d_out_head);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool live = u < deal.turns && u * beside < left;
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"((unsigned)__cvta_generic_to_shared(rstd_slot(stage, u))),
                             "l"(live ? p.rstd + t.row * p.heads + first + u * beside : p.rstd), "r"(live ? 4 : 0)
                             : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    float2 turn[P];
    long long turned = -1;                                      // the row whose angles these are
    long long next_position = 0;
    bool next_good = true;
    int stage = 0;
    if constexpr (RING) {
#pragma unroll
        for (int k = 0; k < kAhead - 1; ++k) copy_ahead(task0 + k, k);
        if (r > 0 && task0 < end) next_good = position_of(a, begin_of(task0).row, flex.table, next_position);
    }
    for (long long task = task0; task < end; task += step) {
        const Begin t = begin_of(task);
        const int n = t.n;
        const b2_heads_part& p = a.part[n];
        const b2_heads_part_grads& d = g.part[n];
        // (heads of the next task are on their way into L2 meanwhile)
        if (!RING && deal.ahead && task + step < end) {
            const Begin t2 = begin_of(task + step);
            const b2_heads_part& p2 = a.part[t2.n];
            const b2_heads_part_grads& d2 = g.part[t2.n];
            const auto fetch = [&](const void* of, long long row_stride, long long head_stride) {
                const T* tensor = static_cast<const T*>(of);
                if constexpr (FLAT) {                       // a lane to a head
                    for (int i = lane; i < each && t2.head + i < a.rows * p2.heads; i += 32) {
                        const long long row = quotient(t2.head + i, p2.heads);
                        const char* at = reinterpret_cast<const char*>(tensor + row * row_stride + (t2.head + i - row * p2.heads) * head_stride);
                        for (int byte = 0; byte < D * (int)sizeof(T); byte += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + byte));
                    }
                } else {                                    // heads next to one another, a lane to 128 bytes
                    if (head_stride != D) return;
                    const char* at = reinterpret_cast<const char*>(tensor + t2.row * row_stride + t2.head * head_stride);
                    const int bytes = min(each, p2.heads - t2.head) * D * (int)sizeof(T);
                    for (int i = lane * 128; i < bytes; i += 32 * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + i));
                }
            };
            fetch(p2.x, p2.x_row, p2.x_head);
            if constexpr (MODE == BACKWARD) fetch(d2.d_out, d2.d_out_row, d2.d_out_head);
        }
        float x[U][N], y[MODE == BACKWARD ? U : 1][N], rstd[U];
        long long position = 0;
        bool good = true;
        // rows and heads of each turn, FLAT; else of the task's first turn
        int row[FLAT ? U : 1] = {}, head[FLAT ? U : 1] = {};
        const auto first = t.head + mine;
        const auto left = (FLAT ? a.rows * p.heads : p.heads) - first;      // heads from this lane's first one on
        if constexpr (FLAT) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (u == 0 || head[u - 1] + beside >= p.heads) {
                    const long long i = first + (u * beside < left ? u * beside : left - 1);       // (of lanes without a head the last one's)
                    row[u] = (int)quotient(i, p.heads);
                    head[u] = (int)(first + u * beside - (long long)row[u] * p.heads);
                } else {
                    row[u] = row[u - 1];
                    head[u] = head[u - 1] + beside;
                }
            }
        }
        // a tensor's head of turn u
        const auto start = [&](auto* tensor, long long row_stride, long long head_stride) { return FLAT ? tensor : tensor + t.row * row_stride + first * head_stride; };
        const auto at_turn = [&](auto* begin, int u, long long row_stride, long long head_stride) {
            if constexpr (FLAT) return begin + (long long)row[u] * row_stride + head[u] * head_stride;
            else return begin + u * beside * head_stride;
        };
        const T* from = start(static_cast<const T*>(p.x), p.x_row, p.x_head);
        const T* from_grad = MODE == BACKWARD ? start(reinterpret_cast<const T*>(d.d_out), d.d_out_row, d.d_out_head) : nullptr;
        if constexpr (RING) {
            copy_ahead(task + kAhead - 1, stage == 0 ? kAhead - 1 : stage - 1);
            position = next_position;
            good = next_good;
            if (r > 0 && task + 1 < end) {
                const long long row2 = begin_of(task + 1).row;
                if (row2 != t.row) next_good = position_of(a, row2, flex.table, next_position);
            }
            asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
        } else if (r > 0 && (FLAT || t.row != turned)) {
            good = position_of(a, FLAT ? row[0] : t.row, flex.table, position);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool live = u < deal.turns && u * beside < left;
            rstd[u] = 1.0f;
            if constexpr (RING) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    get<4>(reinterpret_cast<const float*>(slot_of(stage, 0, u, e)), x[u] + 4 * e);
                    get<4>(reinterpret_cast<const float*>(slot_of(stage, 1, u, e)), y[u] + 4 * e);
                }
                rstd[u] = *reinterpret_cast<const float*>(rstd_slot(stage, u));
            } else if (live) {
                load(at_turn(from, u, p.x_row, p.x_head), x[u]);
                if constexpr (MODE == BACKWARD) {
                    load(at_turn(from_grad, u, d.d_out_row, d.d_out_head), y[u]);
                    rstd[u] = p.rstd[t.row * p.heads + first + u * beside];
                }
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    x[u][j] = 0.0f;
                    if constexpr (MODE == BACKWARD) y[u][j] = 0.0f;
                }
            }
        }
        if constexpr (RING) stage = stage == kAhead - 1 ? 0 : stage + 1;
        float w[N];
        if constexpr (MODE != ROTATE) {
#pragma unroll
            for (int e = 0; e < 2 * EACH; ++e)
                if (p.weight && at[e] >= 0) get<VEC>(p.weight + at[e], w + VEC * e);
                else
#pragma unroll
                    for (int k = 0; k < VEC; ++k) w[VEC * e + k] = 1.0f;
        }
        // the angles of turn u, where its rows are not those of the turn before
        const auto face = [&](int u) {
            if (!FLAT && (u > 0 || t.row == turned)) return;
            turned = t.row;
            if constexpr (FLAT) {
                if (u > 0) {
                    if (!__any_sync(0xffffffffu, row[u] != row[u - 1])) return;
                    if (r > 0) good = position_of(a, row[u], flex.table, position);
                }
            }
#pragma unroll
            for (int k = 0; k < P; ++k) {
                turn[k] = make_float2(1.0f, 0.0f);
                if (r > 0) turn[k] = turn_of((unsigned long long)position * frequency[k], a.amplitude);
                if (!good) turn[k] = make_float2(NAN, NAN);
                if (MODE == BACKWARD || (MODE == ROTATE && a.inverse)) turn[k].y = -turn[k].y;
            }
        };
        T* to = MODE == BACKWARD ? start(reinterpret_cast<T*>(d.d_x), d.d_x_row, d.d_x_head) : start(static_cast<T*>(p.out), p.out_row, p.out_head);
        const auto rotate = [&](float* v) {
            if constexpr (APART) {                              // (a lane's pairs turn all or none)
                if (!turning) return;
#pragma unroll
                for (int k = 0; k < P; k += 2) {
                    const float2 s = two(v + k), t = two(v + VEC + k), c = make_float2(turn[k].x, turn[k + 1].x);
                    apart(__ffma2_rn(t, make_float2(-turn[k].y, -turn[k + 1].y), __fmul2_rn(s, c)), v + k);
                    apart(__ffma2_rn(s, make_float2(turn[k].y, turn[k + 1].y), __fmul2_rn(t, c)), v + VEC + k);
                }
                return;
            }
#pragma unroll
            for (int k = 0; k < P; ++k) {
                if (turning >> k & 1) {
                    const float s = v[2 * k], t = v[2 * k + 1];
                    v[2 * k] = fmaf(s, turn[k].x, -t * turn[k].y);
                    v[2 * k + 1] = fmaf(t, turn[k].x, s * turn[k].y);
                }
            }
        };
        float sum[MODE == BACKWARD ? N : 1];                    // of the task, for its weight
        // sums over the lanes of each head, of all heads next to one another
        const auto over_heads = [&](float (&q)[U]) {
#pragma unroll
            for (int o = 0; o < 5; ++o)
                if (o < deal.lanes)
#pragma unroll
                    for (int u = 0; u < U; ++u) q[u] += __shfl_xor_sync(0xffffffffu, q[u], 1 << o);
        };
        float q[U];
        if constexpr (MODE == FORWARD) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float2 square = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int j = 0; j < N; j += 2) square = __ffma2_rn(two(x[u] + j), two(x[u] + j), square);
                q[u] = square.x + square.y;
            }
            over_heads(q);
        }
        if constexpr (MODE == BACKWARD) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                face(u);
                rotate(y[u]);
                float2 dot = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int j = 0; j < N; j += 2) {
                    const float2 hat = __fmul2_rn(two(x[u] + j), make_float2(rstd[u], rstd[u])), dy = two(y[u] + j), weighted = __fmul2_rn(dy, two(w + j));
                    apart(u == 0 ? __fmul2_rn(dy, hat) : __ffma2_rn(dy, hat, two(sum + j)), sum + j);
                    dot = __ffma2_rn(weighted, hat, dot);
                    apart(hat, x[u] + j);
                    apart(weighted, y[u] + j);
                }
                q[u] = dot.x + dot.y;
            }
            over_heads(q);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u >= deal.turns) break;
            const bool live = u * beside < left;
            float* v = x[u];
            T* out = nullptr;
            if constexpr (MODE == FORWARD) {
                const float root = rsqrtf(fmaf(q[u], share, a.eps));
                if (p.rstd && live && sub == 0) p.rstd[t.row * p.heads + first + u * beside] = root;
#pragma unroll
                for (int j = 0; j < N; j += 2) apart(__fmul2_rn(two(v + j), __fmul2_rn(two(w + j), make_float2(root, root))), v + j);
            }
            if constexpr (MODE == BACKWARD) {
                const float mean = -q[u] * share * rstd[u];
#pragma unroll
                for (int j = 0; j < N; j += 2)
                    apart(__ffma2_rn(two(v + j), make_float2(mean, mean), __fmul2_rn(two(y[u] + j), make_float2(rstd[u], rstd[u]))), v + j);
                if (d.d_x && live) out = at_turn(to, u, d.d_x_row, d.d_x_head);
            } else {
                face(u);
                rotate(v);
                if (live) out = at_turn(to, u, p.out_row, p.out_head);
            }
            if (!out) continue;
            if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int j = 0; j < N; ++j) v[j] *= factor;
                if (flex.probe) {
#pragma unroll
                    for (int j = 0; j < N; ++j) stat = fmaxf(stat, fabsf(v[j]));
                    continue;
                }
            }
#pragma unroll
            for (int e = 0; e < 2 * EACH; ++e)
                if (at[e] >= 0) put<VEC>(out + at[e], v + VEC * e, stat);
        }
        if constexpr (MODE == BACKWARD) {
            if (n) {
#pragma unroll
                for (int j = 0; j < N; ++j) acc[1][j] += sum[j];
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) acc[0][j] += sum[j];
            }
        }
    }
    if constexpr (MODE == BACKWARD) {
        if constexpr (RING) {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncthreads();
        }
        float* words = reinterpret_cast<float*>(table) + (threadIdx.x >> 5) * 2 * D;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2 * EACH; ++e)
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    float q = acc[n][VEC * e + k];
                    for (int o = 1 << deal.lanes; o < 32; o <<= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
                    if (mine == 0 && at[e] >= 0) words[n * D + at[e] + k] = q;
                }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * D; i += kThreads) {
            float v = 0.0f;
#pragma unroll
            for (int k = 0; k < kThreads / 32; ++k) v += reinterpret_cast<const float*>(table)[k * 2 * D + i];
            sums[(long long)blockIdx.x * 2 * D + i] = v;
        }
    }
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) stat = fmaxf(stat, __shfl_xor_sync(0xffffffffu, stat, o));
        if (lane == 0 && stat > 0.0f) {
            if (flex.probe) atomicMax(flex.probe_out, (unsigned long long)__float_as_uint(stat));
            else atomicMax(flex.stats + a.part[0].slot_out, (int)rintf(stat));
        }
    }
}

// Adds the CTAs' sums in their order: a warp to 32 columns and every 32nd CTA, then the warps' sums in their order.
__global__ void __launch_bounds__(1024)
heads_sums_kernel(const float* __restrict__ sums, int ctas, int D, float* d_weight0, float* d_weight1) {
    __shared__ float part[32][33];
    after_earlier_kernels();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = blockIdx.x * 32 + lane;
    float v = 0.0f;
    if (i < 2 * D)
        for (int k = warp; k < ctas; k += 32) v += sums[(long long)k * 2 * D + i];
    part[warp][lane] = v;
    __syncthreads();
    if (warp == 0 && i < 2 * D) {
        v = 0.0f;
        for (int w = 0; w < 32; ++w) v += part[w][lane];
        float* to = i < D ? d_weight0 : d_weight1;
        if (to) to[i < D ? i : i - D] = v;
    }
}

int check_heads(const b2_heads* a, int value_bytes) {
    B2_REQUIRE(a, "missing argument");
    B2_REQUIRE(a->rows >= 0 && a->rows < (1ll << 31), "bad number of rows: %lld", (long long)a->rows);
    B2_REQUIRE(a->head_dim >= 1 && a->head_dim <= kMostDim, "a head has 1 to %d features, not %d", kMostDim, a->head_dim);
    B2_REQUIRE(a->rotary_dim >= 0 && a->rotary_dim <= a->head_dim && a->rotary_dim % 2 == 0, "%d of %d features cannot be rotated", a->rotary_dim,
               a->head_dim);
    B2_REQUIRE(a->parts == 1 || a->parts == 2, "one or two tensors of heads, not %d", a->parts);
    B2_REQUIRE(std::isfinite(a->amplitude) && std::isfinite(a->eps) && a->eps >= 0.0f, "bad amplitude %g or eps %g", a->amplitude, a->eps);
    if (a->rotary_dim > 0) {
        B2_REQUIRE(a->turns && ((uintptr_t)a->turns & 7) == 0, "the frequencies are missing or lie between two addresses");
        B2_REQUIRE(a->position_count >= 1 && a->position_group >= 1, "bad positions: %lld of %lld rows each", (long long)a->position_count,
                   (long long)a->position_group);
        if (a->positions) {
            B2_REQUIRE(a->position_kind >= B2_IDX_F32 && a->position_kind <= B2_IDX_FLEX16, "unknown kind of positions: %d", a->position_kind);
            const uintptr_t size = a->position_kind == B2_IDX_I64 ? 8 : a->position_kind == B2_IDX_FLEX16 ? 2 : 4;
            B2_REQUIRE((uintptr_t)a->positions % size == 0, "a position lies between two addresses");
        }
    }
    for (int i = 0; i < a->parts; ++i) {
        const b2_heads_part& p = a->part[i];
        B2_REQUIRE(p.heads >= 0 && p.heads <= (1 << 20), "bad number of heads: %d", p.heads);
        B2_REQUIRE(((uintptr_t)p.x | (uintptr_t)p.out) % value_bytes == 0 && (((uintptr_t)p.weight | (uintptr_t)p.rstd) & 3) == 0,
                   "a tensor of heads lies between two addresses");
    }
    return B2_OK;
}

// Strides that reach only so far, and for a result no two places for one value.
int check_strides(const b2_heads* a, int heads, int64_t row, int64_t head, bool result, const char* what) {
    if (a->rows == 0 || heads == 0) return B2_OK;
    B2_REQUIRE(row >= 0 && head >= 0 && (a->rows == 1 || row <= (1ll << 46) / a->rows) && (heads == 1 || head <= (1ll << 46) / heads),
               "strides of %s: %lld between rows, %lld between heads", what, (long long)row, (long long)head);
    if (!result) return B2_OK;
    const int64_t D = a->head_dim, across_heads = (heads - 1) * head + D, across_rows = (a->rows - 1) * row + D;
    const bool by_rows = (heads == 1 || head >= D) && (a->rows == 1 || row >= across_heads);
    const bool by_heads = (a->rows == 1 || row >= D) && (heads == 1 || head >= across_rows);
    B2_REQUIRE(by_rows || by_heads, "%s overlaps itself: strides %lld between rows, %lld between heads, %lld features", what, (long long)row, (long long)head,
               (long long)D);
    return B2_OK;
}

// The memory of a tensor of heads.
template <typename T>
Rows heads_at(const T* p, const b2_heads& a, int heads, int64_t row, int64_t head) {
    const long long R = a.rows, D = a.head_dim;
    if (!p || R == 0 || heads == 0) return rows_at(p, 0, 1, 1);
    Rows found = heads == 1                             ? row >= D || R == 1 ? rows_at(p, R, D, row) : rows_at(p, 1, (R - 1) * row + D, D)
                 : R == 1                               ? head >= D ? rows_at(p, heads, D, head) : rows_at(p, 1, (heads - 1) * head + D, D)
                 : head >= D && row == heads * head     ? rows_at(p, R * heads, D, head)
                 : row >= (heads - 1) * head + D        ? rows_at(p, R, (heads - 1) * head + D, row)
                 : head >= (R - 1) * row + D            ? rows_at(p, heads, (R - 1) * row + D, head)
                                                        : rows_at(p, 1, (R - 1) * row + (heads - 1) * head + D, D);
    if (R > 1 && row == 0) return found;                // (one row for all)
    found.at_rows = R;
    found.at_heads = heads;
    found.row_stride = row * (long long)sizeof(T);
    found.head_stride = head * (long long)sizeof(T);
    found.head_width = D * (long long)sizeof(T);
    return found;
}
Rows heads_at(const void* p, const b2_heads& a, int heads, int64_t row, int64_t head, int value_bytes) {
    return value_bytes == 2 ? heads_at(static_cast<const short*>(p), a, heads, row, head) : heads_at(static_cast<const float*>(p), a, heads, row, head);
}
Rows positions_at(const b2_heads& a) {
    if (a.rotary_dim == 0 || !a.positions || a.rows == 0) return rows_at((const char*)nullptr, 0, 0, 0);
    const long long groups = (a.rows + a.position_group - 1) / a.position_group, count = a.position_count < groups ? a.position_count : groups;
    const long long bytes = count * (a.position_kind == B2_IDX_I64 ? 8 : a.position_kind == B2_IDX_FLEX16 ? 2 : 4);
    return rows_at(static_cast<const char*>(a.positions), 1, bytes, bytes);
}
Rows turns_at(const b2_heads& a) { return rows_at(a.rotary_dim ? a.turns : nullptr, 1, a.rotary_dim / 2, a.rotary_dim / 2); }
Rows dense(const float* p, long long n) { return n > 0 ? rows_at(p, 1, n, n) : rows_at(p, 0, 1, 1); }

int check_reads(const b2_heads* a, b2::Memory& memory) {
    if (a->rotary_dim > 0) {
        B2_CHECK(memory.read(a->turns, "the frequencies"));
        B2_CHECK(memory.read(a->positions, "the positions"));
    }
    return B2_OK;
}

int total_heads(const b2_heads& a) { return a.part[0].heads + (a.parts > 1 ? a.part[1].heads : 0); }

// CTAs for heads of any length: rows, and where they are few parts of a row's heads
dim3 grid_any(const b2_heads& a) {
    const long long most = b2::kSms * 16, x = a.rows < most ? a.rows : most;
    long long y = (total_heads(a) + kWarps - 1) / kWarps, room = most / (x > 0 ? x : 1);
    if (y > room) y = room;
    return dim3((unsigned)x, (unsigned)(y < 1 ? 1 : y));
}

// Checks that forward passes share; `sizes` of the values.
int check_forward(const b2_heads* a, int value_bytes, b2::Memory& memory) {
    Rows results[4], operands[6];
    int n = 0, m = 0;
    for (int i = 0; i < a->parts; ++i) {
        const b2_heads_part& p = a->part[i];
        if (p.heads == 0) continue;
        B2_REQUIRE(p.x && p.out, "a tensor of heads is missing");
        B2_CHECK(check_strides(a, p.heads, p.x_row, p.x_head, false, "the heads"));
        B2_CHECK(check_strides(a, p.heads, p.out_row, p.out_head, true, "the result"));
        results[n++] = heads_at(p.out, *a, p.heads, p.out_row, p.out_head, value_bytes);
        if (p.rstd) results[n++] = dense(p.rstd, a->rows * p.heads);
        if (p.x != p.out) operands[m++] = heads_at(p.x, *a, p.heads, p.x_row, p.x_head, value_bytes);
        else B2_REQUIRE((a->rows == 1 || p.x_row == p.out_row) && (p.heads == 1 || p.x_head == p.out_head), "a result in place of its operand has other strides");
        if (p.weight) operands[m++] = dense(p.weight, a->head_dim);
    }
    operands[m++] = positions_at(*a);
    operands[m++] = turns_at(*a);
    B2_CHECK(check_apart(results, n, operands, m, "heads"));
    B2_CHECK(memory.find_device());
    for (int i = 0; i < a->parts; ++i) {
        const b2_heads_part& p = a->part[i];
        if (p.heads == 0) continue;
        B2_CHECK(memory.written(p.out, "the result of heads"));
        if (p.rstd) B2_CHECK(memory.written(p.rstd, "the reciprocal deviations of heads"));
        B2_CHECK(memory.read(p.x, "a tensor of heads"));
        B2_CHECK(memory.read(p.weight, "the weight of heads"));
    }
    return check_reads(a, memory);
}

template <int MODE, typename T>
int launch_any(const b2_heads& a, const b2_heads_grads& g, const FlexArgs& flex, float* sums, dim3 grid, cudaStream_t st) {
    const size_t room = a.rotary_dim / 2 * sizeof(float2) + (MODE == BACKWARD ? kWarps * 2 * a.head_dim * sizeof(float) : 0);
    B2_CUDA((b2::launch_after(heads_any_kernel<MODE, T>, grid, kWarps * 32, room, st, a, g, flex, sums)));
    return B2_OK;
}

// What a launch of heads_kernel deals out, with `runs` lanes wanted by a head and `turns` heads to a lane at once; `flat` receives
// whether by heads: where rows would leave a quarter of the lanes without one, or, `by_heads`, where loads are value by value or from
// page-locked memory.
Deal deal_of(const b2_heads& a, int runs, int turns, bool by_heads, bool* flat) {
    Deal d = {};
    while (d.lanes < 5 && 1 << d.lanes < runs) ++d.lanes;
    const int beside = 32 >> d.lanes;
    const long long heads[2] = {a.part[0].heads, a.parts > 1 ? a.part[1].heads : 0};
    // few heads: one turn to a task, for the least latency
    d.turns = a.rows * (heads[0] + heads[1]) / beside < b2::kSms * 8 ? 1 : turns;
    const long long each = d.turns * beside;
    const long long tasks[2] = {(heads[0] + each - 1) / each, (heads[1] + each - 1) / each};
    *flat = by_heads || (heads[0] + heads[1]) * 4 < (tasks[0] + tasks[1]) * each * 3;
    d.row_tasks = tasks[0] + tasks[1];
    d.first_tasks = *flat ? (a.rows * heads[0] + each - 1) / each : tasks[0];
    d.tasks = *flat ? d.first_tasks + (a.rows * heads[1] + each - 1) / each : a.rows * d.row_tasks;
    d.narrow = a.rows * (heads[0] + heads[1]) < 1ll << 32;
    return d;
}
constexpr int kBackwardCtas = b2::kSms * 3;
int ctas_of(const Deal& d, int mode, int values) {
    const long long all = (d.tasks + kThreads / 32 - 1) / (kThreads / 32), most = stays(mode) ? b2::kSms * blocks_to(mode, values) : 1 << 30;
    return (int)(all < most ? all : most);
}

// Vectors: whole ones of every head lie on 16 bytes, and a run of four features is rotated as a whole or not at all.
bool vectors(const b2_heads& a) { return a.head_dim % 8 == 0 && a.rotary_dim % (a.interleaved ? 4 : 8) == 0; }
bool aligned_heads(const b2_heads& a, const void* p, int64_t row, int64_t head, int heads, int value_bytes) {
    return (uintptr_t)p % (4 * value_bytes) == 0 && (a.rows <= 1 || row % 4 == 0) && (heads <= 1 || head % 4 == 0);
}

template <int MODE, typename T, int VEC, int EACH, bool HALVES, bool FLAT>
int launch_dealt(const b2_heads& a, const b2_heads_grads& g, const FlexArgs& flex, const Deal& deal, float* sums, cudaStream_t st) {
    constexpr bool ring = runs_ahead(MODE, VEC, FLAT);
    const size_t room = ring ? (size_t)kThreads / 32 * kAhead * kSlotBytes : MODE == BACKWARD ? (size_t)kThreads / 32 * 2 * a.head_dim * sizeof(float) : 0;
    static std::atomic<unsigned long long> done{0};
    if (ring) B2_CHECK(b2::allow_shared((const void*)heads_kernel<MODE, T, VEC, EACH, HALVES, FLAT>, (int)room, &done));
    B2_CUDA((b2::launch_after(heads_kernel<MODE, T, VEC, EACH, HALVES, FLAT>, dim3(ctas_of(deal, MODE, 2 * VEC * EACH)), kThreads, room, st, a, g, flex, deal, sums)));
    return B2_OK;
}

// Heads of up to 256 features by heads_kernel, longer ones by heads_any_kernel; `vec`: as vectors; `elsewhere`: operands
// in page-locked memory, which are not fetched ahead.  `ctas` receives how many sums there are.
template <int MODE, typename T>
int launch_heads(const b2_heads& a, const b2_heads_grads& g, const FlexArgs& flex, bool vec, bool elsewhere, float* sums, int* ctas, cudaStream_t st) {
    const int pairs = a.rotary_dim / 2 + (a.head_dim - a.rotary_dim + 1) / 2;
    if (pairs > 128) {
        const dim3 grid = grid_any(a);
        *ctas = (int)(grid.x * grid.y);
        return launch_any<MODE, T>(a, g, flex, sums, grid, st);
    }
    const int runs = vec ? a.head_dim / 8 : pairs, each = vec || runs <= 32 ? 1 : runs <= 64 ? 2 : 4;
    bool flat;
    Deal deal = deal_of(a, runs, unrolled(MODE, vec ? 8 : 2 * each), !vec || elsewhere, &flat);
    deal.ahead = stays(MODE) && !elsewhere;
    *ctas = ctas_of(deal, MODE, vec ? 8 : 2 * each);
#define B2_DEALT(VEC, EACH, FLAT)                                                                                    \
    if (vec == (VEC == 4) && each == EACH && flat == FLAT)                                                           \
        return a.interleaved ? launch_dealt<MODE, T, VEC, EACH, false, FLAT>(a, g, flex, deal, sums, st)             \
                             : launch_dealt<MODE, T, VEC, EACH, true, FLAT>(a, g, flex, deal, sums, st);
    B2_DEALT(4, 1, false)
    B2_DEALT(4, 1, true)
    B2_DEALT(1, 1, true)
    B2_DEALT(1, 2, true)
    B2_DEALT(1, 4, true)
#undef B2_DEALT
    return b2::fail(B2_ERR_INVALID, "no kernel for heads of %d features", a.head_dim);
}

bool forward_vectors(const b2_heads& a, int value_bytes) {
    bool vec = vectors(a);
    for (int i = 0; i < a.parts; ++i) {
        const b2_heads_part& p = a.part[i];
        vec = vec && (p.heads == 0 || (aligned_heads(a, p.x, p.x_row, p.x_head, p.heads, value_bytes) && aligned_heads(a, p.out, p.out_row, p.out_head, p.heads, value_bytes) &&
                                       b2::aligned16(p.weight)));
    }
    return vec;
}

}  // namespace

extern "C" int b2_rotary_turns(int32_t rotary_dim, double base, int32_t scaling, double factor, double original, double low, double high, uint64_t* turns) {
    B2_REQUIRE(rotary_dim >= 0 && rotary_dim <= kMostDim && rotary_dim % 2 == 0, "%d features cannot be rotated", rotary_dim);
    B2_REQUIRE(turns || rotary_dim == 0, "missing argument");
    B2_REQUIRE(std::isfinite(base) && base > 0.0, "bad base: %g", base);
    B2_REQUIRE(scaling >= B2_ROTARY_PLAIN && scaling <= B2_ROTARY_PARTS, "unknown scaling: %d", scaling);
    B2_REQUIRE(scaling == B2_ROTARY_PLAIN || (std::isfinite(factor) && factor > 0.0), "bad factor: %g", factor);
    B2_REQUIRE(scaling != B2_ROTARY_PARTS || (std::isfinite(original) && original > 0.0 && std::isfinite(low) && std::isfinite(high) && low < high),
               "bad parts: context %g, from %g to %g turns", original, low, high);
    // (64 bits of a fraction want a significand of 64 bits: angles by frequencies of doubles are off by 2^-36 of a turn at position a million)
    static_assert(std::numeric_limits<long double>::digits >= 64, "frequencies have 64 bits");
    const long double d = rotary_dim, circle = 6.28318530717958647692528676655900577L, by = factor;
    long double from = base;
    if (scaling == B2_ROTARY_BASE && rotary_dim > 2) from *= std::pow(by, d / (d - 2));
    for (int i = 0; i < rotary_dim / 2; ++i) {
        long double f = std::pow(from, -2.0L * i / d) / circle;     // turns a position
        if (scaling == B2_ROTARY_LINEAR) f /= by;
        if (scaling == B2_ROTARY_PARTS) {
            long double keep = (original * f - low) / ((long double)high - low);
            keep = keep < 0.0L ? 0.0L : keep > 1.0L ? 1.0L : keep;
            f = keep * f + (1.0L - keep) * f / by;
        }
        B2_REQUIRE(std::isfinite((double)f), "frequency %d is not finite", i);
        f -= std::floor(f);
        // (a value just below one may round to a whole turn)
        const long double whole = std::nearbyint(f * 18446744073709551616.0L);
        turns[i] = whole >= 18446744073709551616.0L ? 0 : (uint64_t)whole;
    }
    return B2_OK;
}

extern "C" int b2_rotary(const b2_heads* a, int32_t flex, const b2_flex_scale* scales, int32_t* stats, uint64_t* probe_out, int32_t probe, void* stream) {
    const int size = flex ? 2 : 4;
    B2_CHECK(check_heads(a, size));
    for (int i = 0; i < a->parts; ++i) B2_REQUIRE(!a->part[i].weight && !a->part[i].rstd, "a weight or deviations without a norm");
    B2_REQUIRE(flex || a->rotary_dim == 0 || !a->positions || a->position_kind != B2_IDX_FLEX16 || scales, "flex16 positions have an exponent");
    if (flex) {
        B2_REQUIRE(a->parts == 1, "one tensor in flex16, not %d", a->parts);
        B2_REQUIRE(scales && a->part[0].slot_x >= 0 && a->part[0].slot_out >= 0 && (probe ? probe_out != nullptr : stats != nullptr), "missing exponents or statistics");
    }
    B2_REQUIRE(a->rotary_dim == 0 || !a->positions || a->position_kind != B2_IDX_FLEX16 || a->slot_positions >= 0, "flex16 positions have an exponent");
    B2_REQUIRE((((uintptr_t)scales | (uintptr_t)stats) & 3) == 0 && ((uintptr_t)probe_out & 7) == 0, "exponents or statistics lie between two addresses");
    if (a->rows == 0 || total_heads(*a) == 0) return B2_OK;
    b2::Memory memory;
    B2_CHECK(check_forward(a, size, memory));
    const FlexArgs f = {scales, stats, (unsigned long long*)probe_out, probe};
    const bool scaled = flex || (a->positions && a->position_kind == B2_IDX_FLEX16);
    if (scaled) B2_CHECK(memory.read(scales, "the exponents"));
    if (flex) B2_CHECK(probe ? memory.written(probe_out, "the largest value") : memory.written(stats, "the statistics"));
    cudaStream_t st = (cudaStream_t)stream;
    int ctas;
    if (flex) return launch_heads<ROTATE, short>(*a, b2_heads_grads{}, f, forward_vectors(*a, 2), memory.elsewhere, nullptr, &ctas, st);
    return launch_heads<ROTATE, float>(*a, b2_heads_grads{}, f, forward_vectors(*a, 4), memory.elsewhere, nullptr, &ctas, st);
}

static int check_norm_of_heads(const b2_heads* a) {
    B2_CHECK(check_heads(a, 4));
    B2_REQUIRE(!a->inverse, "a norm's rotation is not turned back: its gradient does that itself");
    B2_REQUIRE(a->rotary_dim == 0 || !a->positions || a->position_kind != B2_IDX_FLEX16, "flex16 positions of fp32 heads");
    return B2_OK;
}

extern "C" int b2_heads_fprop(const b2_heads* a, void* stream) {
    B2_CHECK(check_norm_of_heads(a));
    if (a->rows == 0 || total_heads(*a) == 0) return B2_OK;
    b2::Memory memory;
    B2_CHECK(check_forward(a, 4, memory));
    int ctas;
    return launch_heads<FORWARD, float>(*a, b2_heads_grads{}, FlexArgs{}, forward_vectors(*a, 4), memory.elsewhere, nullptr, &ctas, (cudaStream_t)stream);
}

extern "C" int b2_heads_bprop_scratch_bytes(const b2_heads* a, size_t* bytes) {
    B2_REQUIRE(bytes, "missing argument");
    B2_CHECK(check_norm_of_heads(a));
    const dim3 grid = grid_any(*a);
    const size_t ctas = (size_t)grid.x * grid.y;
    *bytes = (ctas > kBackwardCtas ? ctas : kBackwardCtas) * 2 * a->head_dim * sizeof(float) + 256;
    return B2_OK;
}

extern "C" int b2_heads_bprop(const b2_heads* a, const b2_heads_grads* g, void* scratch, size_t scratch_bytes, void* stream) {
    size_t need = 0;
    B2_CHECK(b2_heads_bprop_scratch_bytes(a, &need));
    B2_REQUIRE(g, "missing argument");
    B2_REQUIRE(scratch && scratch_bytes >= need, "the gradient of heads needs %zu bytes of scratch, got %zu", need, scratch_bytes);
    Rows results[5], operands[10];
    int n = 0, m = 0;
    float* weights[2] = {nullptr, nullptr};
    results[n++] = rows_at((const char*)scratch, 1, (long long)need, (long long)need);
    for (int i = 0; i < a->parts; ++i) {
        const b2_heads_part& p = a->part[i];
        const b2_heads_part_grads& d = g->part[i];
        B2_REQUIRE((((uintptr_t)d.d_out | (uintptr_t)d.d_x | (uintptr_t)d.d_weight) & 3) == 0, "a gradient of heads lies between two addresses");
        B2_REQUIRE(p.weight || !d.d_weight, "the gradient of a weight that is not there");
        weights[i] = d.d_weight;
        if (d.d_weight) results[n++] = dense(d.d_weight, a->head_dim);
        if (p.weight) operands[m++] = dense(p.weight, a->head_dim);
        if (a->rows == 0 || p.heads == 0) continue;
        B2_REQUIRE(p.x && p.rstd && d.d_out, "the gradient of heads reads x, rstd and d_out");
        B2_CHECK(check_strides(a, p.heads, p.x_row, p.x_head, false, "the heads"));
        B2_CHECK(check_strides(a, p.heads, d.d_out_row, d.d_out_head, false, "the result's gradient"));
        operands[m++] = heads_at((const float*)p.x, *a, p.heads, p.x_row, p.x_head);
        operands[m++] = dense(p.rstd, a->rows * p.heads);
        if (d.d_x) {
            B2_CHECK(check_strides(a, p.heads, d.d_x_row, d.d_x_head, true, "the heads' gradient"));
            results[n++] = heads_at((const float*)d.d_x, *a, p.heads, d.d_x_row, d.d_x_head);
            B2_REQUIRE(d.d_x != d.d_out || ((a->rows == 1 || d.d_x_row == d.d_out_row) && (p.heads == 1 || d.d_x_head == d.d_out_head)),
                       "a gradient in place of its operand has other strides");
        }
        if (d.d_x != d.d_out) operands[m++] = heads_at(d.d_out, *a, p.heads, d.d_out_row, d.d_out_head);
    }
    operands[m++] = positions_at(*a);
    operands[m++] = turns_at(*a);
    B2_CHECK(check_apart(results, n, operands, m, "heads' gradient"));
    b2::Memory memory;
    B2_CHECK(memory.find_device());
    B2_CHECK(memory.written(scratch, "the scratch of heads"));
    const bool work = a->rows > 0 && total_heads(*a) > 0;
    for (int i = 0; i < a->parts; ++i) {
        const b2_heads_part& p = a->part[i];
        const b2_heads_part_grads& d = g->part[i];
        if (d.d_weight) B2_CHECK(memory.written(d.d_weight, "the gradient of a weight"));
        B2_CHECK(memory.read(p.weight, "the weight of heads"));
        if (!work || p.heads == 0) continue;
        if (d.d_x) B2_CHECK(memory.written(d.d_x, "the gradient of heads"));
        B2_CHECK(memory.read(p.x, "a tensor of heads"));
        B2_CHECK(memory.read(p.rstd, "the reciprocal deviations of heads"));
        B2_CHECK(memory.read(d.d_out, "the gradient of a result"));
    }
    if (work) B2_CHECK(check_reads(a, memory));
    cudaStream_t st = (cudaStream_t)stream;
    float* sums = (float*)(((uintptr_t)scratch + 255) / 256 * 256);
    bool vec = vectors(*a);
    for (int i = 0; i < a->parts; ++i) {
        const b2_heads_part& p = a->part[i];
        const b2_heads_part_grads& d = g->part[i];
        vec = vec && (p.heads == 0 || (aligned_heads(*a, p.x, p.x_row, p.x_head, p.heads, 4) && aligned_heads(*a, d.d_out, d.d_out_row, d.d_out_head, p.heads, 4) &&
                                       (!d.d_x || aligned_heads(*a, d.d_x, d.d_x_row, d.d_x_head, p.heads, 4)) && b2::aligned16(p.weight)));
    }
    int ctas = 0;
    if (work) B2_CHECK((launch_heads<BACKWARD, float>(*a, *g, FlexArgs{}, vec, memory.elsewhere, sums, &ctas, st)));
    if (weights[0] || weights[1]) {
        const int D = a->head_dim;
        B2_CUDA((b2::launch_after(heads_sums_kernel, dim3((2 * D + 31) / 32), 1024, 0, st, (const float*)sums, ctas, D,
                                  weights[0], weights[1])));
    }
    return B2_OK;
}
