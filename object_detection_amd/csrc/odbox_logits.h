// odbox_logits.h -- what the two units of the class-logit operators share: element types, the arguments of the kernels, and how
// the kernels for short rows (odbox_logits_short.hip) are reached from the entry points (odbox_logits.hip).
#ifndef ODBOX_LOGITS_H
#define ODBOX_LOGITS_H
#include "odbox_common.h"

namespace odbox {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN2 = 0.69314718055994530942f;
constexpr float T_FLOOR = -16384.0f;             // stands for log2 p = -inf in p * log2 p (2^-16384 is 0, so the product is 0)
constexpr float M_START = -1e30f;                // a running maximum before any class; times c it is still finite

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

// Element types: 16-byte vectors that may start at any element (rows of an odd number of classes do: global_load / store_dwordx4
// take any alignment).  Stores round to nearest even.
template <class V, int ALIGN>
struct Unaligned {
    typedef V type __attribute__((aligned(ALIGN)));
};
struct F32 {
    using raw = float;
    static __device__ __forceinline__ u32x4 none() { return u32x4{0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u}; }   // -inf
    static constexpr int VEC = 4;
    static __device__ __forceinline__ float get(raw v) { return v; }
    static __device__ __forceinline__ raw put(float v) { return v; }
    static __device__ __forceinline__ void unpack(u32x4 w, float *v)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
    }
    static __device__ __forceinline__ u32x4 pack(const float *v)
    {
        return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    }
};
struct F16 {
    using raw = _Float16;
    static __device__ __forceinline__ u32x4 none() { return u32x4{0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u}; }
    static constexpr int VEC = 8;
    static __device__ __forceinline__ float get(raw v) { return (float)v; }
    static __device__ __forceinline__ raw put(float v) { return (_Float16)v; }
    // the 16 bits of a value as an unsigned number of the same order (-0 folded into +0, NaN above all), and back
    static __device__ __forceinline__ uint32_t order16(float v)
    {
        const uint32_t u = __builtin_bit_cast(uint16_t, (_Float16)(v + 0.0f));
        return v != v ? 0xffffu : u & 0x8000u ? u ^ 0xffffu : u | 0x8000u;
    }
    static __device__ __forceinline__ float value16(uint32_t o)
    {
        return o == 0xffffu ? NAN : (float)__builtin_bit_cast(_Float16, (uint16_t)(o & 0x8000u ? o & 0x7fffu : o ^ 0xffffu));
    }
    static __device__ __forceinline__ void unpack(u32x4 w, float *v)
    {
        const f16x8 h = __builtin_bit_cast(f16x8, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
    }
    static __device__ __forceinline__ u32x4 pack(const float *v)
    {
        f16x8 h;
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = (_Float16)v[i];
        return __builtin_bit_cast(u32x4, h);
    }
};
struct BF16 {
    using raw = uint16_t;
    static __device__ __forceinline__ u32x4 none() { return u32x4{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u}; }
    static constexpr int VEC = 8;
    static __device__ __forceinline__ float get(raw v) { return __uint_as_float((uint32_t)v << 16); }
    static __device__ __forceinline__ raw put(float v) { return __builtin_bit_cast(raw, (__bf16)v); }
    static __device__ __forceinline__ uint32_t order16(float v) { return v != v ? 0xffffu : f32_ordered(v) >> 16; }
    static __device__ __forceinline__ float value16(uint32_t o)
    {
        return o == 0xffffu ? NAN : __uint_as_float((o & 0x8000u ? o & 0x7fffu : o ^ 0xffffu) << 16);
    }
    static __device__ __forceinline__ void unpack(u32x4 w, float *v)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float *v)
    {
        f32x8 f;
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = v[i];
        return __builtin_bit_cast(u32x4, __builtin_convertvector(f, bf16x8));
    }
};
// PASSING: data that passes by once goes around the caches.
template <class E, bool PASSING = false>
__device__ __forceinline__ u32x4 load_raw(const typename E::raw *p)
{
    typedef typename Unaligned<u32x4, sizeof(typename E::raw)>::type mem;
    return PASSING ? __builtin_nontemporal_load((const mem *)p) : *(const mem *)p;
}
template <class E, bool PASSING = false>
__device__ __forceinline__ void store_raw(typename E::raw *p, u32x4 v)
{
    typedef typename Unaligned<u32x4, sizeof(typename E::raw)>::type mem;
    if (PASSING) __builtin_nontemporal_store(v, (mem *)p);
    else *(mem *)p = v;
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_hw(float x) { return __builtin_amdgcn_logf(x); }
__device__ __forceinline__ float vmax3(float a, float b, float c)
{
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_f(float old, float x)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(x), CTRL, ROWS, 0xf, false));
}
// x of the wave's lanes combined in lane 63 and handed to all; `none` is the operation's neutral value
template <class Op>
__device__ __forceinline__ float wave_reduce(float x, float none, Op op)
{
    x = op(x, dpp_f<0x111, 0xf>(none, x));       // row_shr:1
    x = op(x, dpp_f<0x112, 0xf>(none, x));       // row_shr:2
    x = op(x, dpp_f<0x114, 0xf>(none, x));       // row_shr:4
    x = op(x, dpp_f<0x118, 0xf>(none, x));       // row_shr:8
    x = op(x, dpp_f<0x142, 0xa>(none, x));       // row_bcast:15 into rows 1 and 3
    x = op(x, dpp_f<0x143, 0xc>(none, x));       // row_bcast:31 into rows 2 and 3
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}
__device__ __forceinline__ float wave_max(float x) { return wave_reduce(x, -INFINITY, [](float a, float b) { return vmax(a, b); }); }
__device__ __forceinline__ float wave_sum(float x) { return wave_reduce(x, 0.0f, [](float a, float b) { return a + b; }); }

struct RowStats {
    float m;             // largest logit; -inf: every logit is -inf (an empty row); NaN: the row holds a NaN or +inf
    float l2;            // log2 of the sum
    float ent;           // entropy in nats
    float s;             // the sum itself
};

struct ScoreArgs {
    const void *logits;
    size_t rows, stride;
    uint32_t C, k;
    float c, inv_t;
    const int32_t *labels;
    float *logprobs, *entropy, *top_logprobs;
    int32_t *top_labels;
    float4 *stats;
    uint32_t segs, seg;                          // a row's classes go to `segs` blocks, `seg` (a multiple of 8) to each
    float4 *part;                                // [rows, segs] shares of a split row
    uint64_t *part_key;                          // [rows, segs, k]
};

template <class E>
__device__ __forceinline__ float logprob_of(const ScoreArgs &a, const RowStats &st, float v)
{
    return st.m == -INFINITY ? -INFINITY : (v - st.m) * a.inv_t - LN2 * st.l2;
}

struct ScoreGradArgs {
    const void *logits;
    size_t rows, stride;
    uint32_t C, k;
    float c, inv_t;
    const int32_t *labels, *top_labels;
    const float4 *stats;
    const float *up_logprobs, *up_entropy, *up_top;
    void *grad;
    uint32_t segs, seg;
};

struct DistillArgs {
    const void *logits;
    size_t rows, stride;
    uint32_t C, K;
    float c, t, inv_t, scale;
    int bucket;
    const float *teacher;
    const int32_t *ids;
    const float *weights;
    float *out_rows;
    float4 *stats;
    const float *up;
    int up_rows;
    void *grad;
    uint32_t segs, seg;
    float4 *part;                                // [rows, segs] shares of a split row
};

// exp(t) to about 2^-23 relative for t <= 0: the product with log2(e) in two parts
__device__ __forceinline__ float exp_split(float t)
{
    const float hi = t * LOG2E;
    if (!(hi > -150.0f)) return t != t ? t : 0.0f;
    const float lo = __builtin_fmaf(t, LOG2E, -hi) + t * 1.925963033500e-08f;      // LOG2E is log2(e) less that
    return exp2_hw(hi) * __builtin_fmaf(lo, LN2, 1.0f);
}

// exp(t) for t <= 0 to 2^-51 absolute, for sums that are taken from 1: 2^k exp(r)^2 with |2 r| <= ln(2) / 2, exp(r) by its series up to
// r^10 / 10! (r^11 / 11! < 2^-53); below -40 it is 0, which is 2^-57 off.  The coefficients are handed over in scalar registers: held from row
// to row in vector registers, as the compiler and the library's exponential do, they cost the row its own (bucket losses of 2048 x
// 32768 34 -> 47 us).
__device__ __forceinline__ double exp_wide(float t)
{
    if (!(t > -40.0f)) return t != t ? (double)t : 0.0;
    const float k = __builtin_rintf(t * LOG2E);
    const double r = __builtin_fma((double)k, -0.69314718055994530942 / 2, (double)t * 0.5);
    double e = 1.0 / 3628800;
    const auto step = [&](double c) {
        asm volatile("" : "+s"(c));
        e = __builtin_fma(e, r, c);
    };
    asm volatile("" : "+s"(e));
    step(1.0 / 362880);
    step(1.0 / 40320);
    step(1.0 / 5040);
    step(1.0 / 720);
    step(1.0 / 120);
    step(1.0 / 24);
    step(1.0 / 6);
    e = __builtin_fma(e, r, 0.5);
    e = __builtin_fma(e, r, 1.0);
    e = __builtin_fma(e, r, 1.0);
    return __builtin_ldexp(e * e, (int)k);
}

// log(1 + x) for |x| <= 1/2 or 0 <= x <= 1, as exact near 0 as elsewhere: the rounding of 1 + x is taken out by x / ((1 + x) - 1)
__device__ __forceinline__ float log1p_hw(float x)
{
    const float u = 1.0f + x;
    return u == 1.0f ? x : LN2 * log2_hw(u) * (x / (u - 1.0f));
}

// The bucket of a row: p0 and q0, the student's and the teacher's mass off the list.  Where the list holds little both are near 1, and loss and
// gradient live on their difference: there they come from on / off and sum q, which are small, and not from what those leave of 1.
struct BucketTerms {
    float dense;         // p0 (sum q + q0) - q0
    float rest;          // q0 (log q0 - log p0)
};
// on, off: the student's sums on and off the list; log_far: log p0 from maxima and logarithms, for a p0 that float32 does not reach
__device__ __forceinline__ BucketTerms bucket_terms(float on, float off, float sum_q, float q0, float log_far)
{
    const float s = on + off, p0 = off / s;
    BucketTerms r;
    r.dense = q0 > 0.0f && p0 > 0.5f ? sum_q - on / s : p0 * (sum_q + q0) - q0;
    const float log_q0 = sum_q < 0.5f ? log1p_hw(-sum_q) : LN2 * log2_hw(q0);
    const float log_p0 = p0 > 0.5f ? -log1p_hw(on / off) : p0 > 1e-30f ? LN2 * log2_hw(p0) : log_far;
    r.rest = q0 > 0.0f ? q0 * (log_q0 - log_p0) : 0.0f;
    return r;
}

#define LOGITS_LAUNCH(dtype, K_, ...)                                                       \
    do {                                                                                    \
        if ((dtype) == ODBOX_DTYPE_F32) { using E = F32; hipLaunchKernelGGL(K_, __VA_ARGS__); } \
        else if ((dtype) == ODBOX_DTYPE_F16) { using E = F16; hipLaunchKernelGGL(K_, __VA_ARGS__); } \
        else { using E = BF16; hipLaunchKernelGGL(K_, __VA_ARGS__); }                        \
    } while (0)

inline dim3 work_grid(size_t work) { return dim3((uint32_t)(work < 1u << 20 ? work : 1u << 20)); }

// Rows short enough for the registers of a few lanes (odbox_logits_short.hip); each launches one kernel on st.
int short_limit(int dtype);                      // classes
bool score_is_short(int dtype, int C, int k);
void score_short(int dtype, const ScoreArgs &a, hipStream_t st);
void score_grad_short(int dtype, const ScoreGradArgs &a, hipStream_t st);
void distill_short(int dtype, int rest, bool grad, const DistillArgs &a, hipStream_t st);

}  // namespace odbox
#endif
