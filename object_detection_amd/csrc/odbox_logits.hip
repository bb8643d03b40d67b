// odbox_logits.hip -- operators on rows of class logits: log-probabilities of given labels with entropy and top
// alternatives, and distillation from a teacher's top classes, forward and backward.  No counterpart in the reference,
// whose only softmax is metric.py:19-20; the entry points stand beside odbox_focal_loss_rows.
//
// Notation of every kernel here: a row x of C logits, c = log2(e) / temperature, m = the row's largest logit,
// s = sum 2^((x - m) c), l2 = log2(s); log2 p_i = (x_i - m) c - l2.  m is taken out BEFORE the multiplication, so that rows
// of large or shifted logits lose nothing; log-probabilities that are returned are (x_i - m) / T - ln2 l2, which stays finite as
// far as float32 reaches.  Sums, maxima and outputs other than gradients are 32-bit floats.
#include "odbox_common.h"

namespace odbox {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN2 = 0.69314718055994530942f;
constexpr float T_FLOOR = -16384.0f;             // stands for log2 p = -inf in p * log2 p (2^-16384 is 0, so the product is 0)
constexpr int LG_THREADS = 256;
constexpr int LG_WAVES = LG_THREADS / WAVE;

struct F32 {
    using raw = float;
    static __device__ __forceinline__ float get(raw v) { return v; }
    static __device__ __forceinline__ raw put(float v) { return v; }
};
struct F16 {
    using raw = _Float16;
    static __device__ __forceinline__ float get(raw v) { return (float)v; }
    static __device__ __forceinline__ raw put(float v) { return (_Float16)v; }
};
struct BF16 {
    using raw = uint16_t;
    static __device__ __forceinline__ float get(raw v) { return __uint_as_float((uint32_t)v << 16); }
    // round to nearest even; a NaN keeps its sign and becomes quiet (the carry of the rounding must not turn it into inf)
    static __device__ __forceinline__ raw put(float v)
    {
        const uint32_t u = __float_as_uint(v);
        if ((u & 0x7fffffffu) > 0x7f800000u) return (raw)((u >> 16) | 0x40u);
        return (raw)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
    }
};

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_hw(float x) { return __builtin_amdgcn_logf(x); }

// What one block shares: wave partials of the reductions, the radix histogram, the chosen keys.
struct LogitsLds {
    double d[LG_WAVES];
    float f[LG_WAVES];
    uint32_t hist[256];
    uint64_t key[ODBOX_MAX_TOP];
    uint32_t count;
    uint32_t pick[2];
    int32_t id[ODBOX_MAX_TOP + 1];
    float val[ODBOX_MAX_TOP + 1];
};

template <class Op>
__device__ __forceinline__ float block_reduce(float v, LogitsLds &sh, Op op)
{
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = op(v, __shfl_xor(v, off));
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) sh.f[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh.f[0];
#pragma unroll
    for (int w = 1; w < LG_WAVES; ++w) v = op(v, sh.f[w]);
    return v;
}
__device__ __forceinline__ float block_max(float v, LogitsLds &sh) { return block_reduce(v, sh, [](float a, float b) { return vmax(a, b); }); }
__device__ __forceinline__ float block_sum(float v, LogitsLds &sh) { return block_reduce(v, sh, [](float a, float b) { return a + b; }); }
__device__ __forceinline__ double block_sum_f64(double v, LogitsLds &sh)
{
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) sh.d[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh.d[0];
#pragma unroll
    for (int w = 1; w < LG_WAVES; ++w) v += sh.d[w];
    return v;
}

struct RowStats {
    float m;             // largest logit; -inf: every logit is -inf (an empty row); NaN: the row holds a NaN or +inf
    float l2;            // log2 of the sum
    float ent;           // entropy in nats
};

// Two passes over the row by the whole block.  skip(i): class i is left out.
template <class E, class Skip>
__device__ RowStats row_stats(const typename E::raw *x, uint32_t C, float c, LogitsLds &sh, Skip skip)
{
    float m = -INFINITY, bad = 0.0f;
    for (uint32_t i = threadIdx.x; i < C; i += LG_THREADS) {
        const float v = E::get(x[i]);
        if (skip(i)) continue;
        if (v != v || v == INFINITY) bad = 1.0f;
        m = vmax(m, v);
    }
    m = block_max(m, sh);
    bad = block_max(bad, sh);
    if (bad != 0.0f) return {NAN, NAN, NAN};
    if (m == -INFINITY) return {m, -INFINITY, 0.0f};
    float s = 0.0f, u = 0.0f;
    for (uint32_t i = threadIdx.x; i < C; i += LG_THREADS) {
        if (skip(i)) continue;
        const float t = (E::get(x[i]) - m) * c, e = exp2_hw(t);
        s += e;
        u += e * vmax(t, T_FLOOR);
    }
    s = block_sum(s, sh);
    u = block_sum(u, sh);
    const float l2 = log2_hw(s);
    return {m, l2, LN2 * (l2 - u / s)};
}

// Order of the top alternatives: value descending, then index ascending; NaN above everything.  56 significant bits.
__device__ __forceinline__ uint64_t top_key(float v, uint32_t i)
{
    const uint32_t o = v != v ? 0xffffffffu : f32_ordered(v);
    return ((uint64_t)o << 24) | (0xffffffu - i);
}
__device__ __forceinline__ uint32_t top_index(uint64_t k) { return 0xffffffu - ((uint32_t)k & 0xffffffu); }

// The k (<= ODBOX_MAX_TOP, <= n) largest of n unique keys into sh.key, ordered descending: the k-th key by a radix selection of
// eight bits a pass, then exactly k keys are collected and each counts those above it.
template <class Key>
__device__ void top_radix(uint32_t n, uint32_t k, LogitsLds &sh, Key key)
{
    uint64_t prefix = 0;
    uint32_t want = k;
    for (int shift = 48; shift >= 0; shift -= 8) {
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < 256; i += LG_THREADS) sh.hist[i] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < n; i += LG_THREADS) {
            const uint64_t q = key(i);
            if ((q >> shift >> 8) == prefix) atomicAdd(&sh.hist[(uint32_t)(q >> shift) & 255u], 1u);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            uint32_t above = 0, b = 255;
            while (b > 0 && above + sh.hist[b] < want) above += sh.hist[b--];
            sh.pick[0] = b;
            sh.pick[1] = above;
        }
        __syncthreads();
        prefix = (prefix << 8) | sh.pick[0];
        want -= sh.pick[1];
    }
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    uint64_t mine = 0;
    for (uint32_t i = threadIdx.x; i < n; i += LG_THREADS) {
        const uint64_t q = key(i);
        if (q >= prefix) sh.key[atomicAdd(&sh.count, 1u)] = q;        // unique keys: exactly k of them
    }
    __syncthreads();
    uint32_t rank = 0;
    if (threadIdx.x < k) {
        mine = sh.key[threadIdx.x];
        for (uint32_t j = 0; j < k; ++j) rank += sh.key[j] > mine;
    }
    __syncthreads();
    if (threadIdx.x < k) sh.key[rank] = mine;
    __syncthreads();
}

struct ScoreArgs {
    const void *logits;
    size_t rows, stride;
    uint32_t C, k;
    float c, inv_t;
    const int32_t *labels;
    float *logprobs, *entropy, *top_logprobs;
    int32_t *top_labels;
    float4 *stats;
};

template <class E>
__global__ __launch_bounds__(LG_THREADS) void score_rows_kernel(ScoreArgs a)
{
    __shared__ LogitsLds sh;
    for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const typename E::raw *x = (const typename E::raw *)a.logits + row * a.stride;
        const RowStats st = row_stats<E>(x, a.C, a.c, sh, [](uint32_t) { return false; });
        auto logprob = [&](float v) { return st.m == -INFINITY ? -INFINITY : (v - st.m) * a.inv_t - LN2 * st.l2; };
        if (threadIdx.x == 0) {
            if (a.logprobs) {
                const uint32_t lab = (uint32_t)a.labels[row];
                a.logprobs[row] = lab < a.C ? logprob(E::get(x[lab])) : 0.0f;
            }
            if (a.entropy) a.entropy[row] = st.ent;
            if (a.stats) a.stats[row] = make_float4(st.m, st.l2, st.ent, 0.0f);
        }
        if (a.k) {
            top_radix(a.C, a.k, sh, [&](uint32_t i) { return top_key(E::get(x[i]), i); });
            if (threadIdx.x < a.k) {
                const uint32_t i = top_index(sh.key[threadIdx.x]);
                a.top_labels[row * a.k + threadIdx.x] = (int32_t)i;
                a.top_logprobs[row * a.k + threadIdx.x] = logprob(E::get(x[i]));
            }
            __syncthreads();
        }
    }
}

// What the gradient of a row looks like: scale * p_i * (a + b * log2 p_i) everywhere (p of the streamed classes), and at the
// n listed classes id[] the values val[], which are final.
struct RowGrad {
    float m, l2, a, b;
    uint32_t n;
};

struct ScoreGradArgs {
    const void *logits;
    size_t rows, stride;
    uint32_t C, k;
    float c, inv_t;
    const int32_t *labels, *top_labels;
    const float4 *stats;
    const float *up_logprobs, *up_entropy, *up_top;
    void *grad;
};

// A class that is listed twice gets the sum of its entries; only its first entry writes.
__device__ __forceinline__ bool first_entry(const LogitsLds &sh, uint32_t j, uint32_t n, float &sum)
{
    const int32_t id = sh.id[j];
    sum = 0.0f;
    for (uint32_t i = 0; i < n; ++i) {
        if (sh.id[i] != id) continue;
        if (i < j) return false;
        sum += sh.val[i];
    }
    return true;
}

template <class E>
__device__ void write_grad(const RowGrad &g, const typename E::raw *x, typename E::raw *out, uint32_t C, float c, LogitsLds &sh)
{
    const bool none = g.m == -INFINITY;                      // no streamed class has any probability
    for (uint32_t i = threadIdx.x; i < C; i += LG_THREADS) {
        const float t = (E::get(x[i]) - g.m) * c - g.l2;
        out[i] = E::put(none ? 0.0f : exp2_hw(t) * (g.a + g.b * vmax(t, T_FLOOR)));
    }
    __syncthreads();                                         // the block's own stores before the listed classes' (same addresses)
    for (uint32_t j = threadIdx.x; j < g.n; j += LG_THREADS)
        if (sh.id[j] >= 0) out[sh.id[j]] = E::put(sh.val[j]);
    __syncthreads();
}

template <class E>
__global__ __launch_bounds__(LG_THREADS) void score_grad_kernel(ScoreGradArgs a)
{
    __shared__ LogitsLds sh;
    for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const typename E::raw *x = (const typename E::raw *)a.logits + row * a.stride;
        typename E::raw *out = (typename E::raw *)a.grad + row * a.C;
        const float4 st = a.stats[row];
        if (st.x == -INFINITY) {                             // an empty row has constant outputs
            for (uint32_t i = threadIdx.x; i < a.C; i += LG_THREADS) out[i] = E::put(0.0f);
            continue;
        }
        const uint32_t n = a.k + 1;
        const float gh = a.up_entropy ? a.up_entropy[row] : 0.0f;
        __syncthreads();
        for (uint32_t j = threadIdx.x; j < n; j += LG_THREADS) {
            int32_t id = -1;
            float v = 0.0f;
            if (j == a.k) {
                if (a.up_logprobs && (uint32_t)a.labels[row] < a.C) id = a.labels[row], v = a.up_logprobs[row];
            } else if (a.up_top)
                id = a.top_labels[row * a.k + j], v = a.up_top[row * a.k + j];
            sh.id[j] = (uint32_t)id < a.C ? id : -1;
            sh.val[j] = (uint32_t)id < a.C ? v : 0.0f;
        }
        __syncthreads();
        float part = 0.0f;
        for (uint32_t j = threadIdx.x; j < n; j += LG_THREADS) part += sh.val[j];
        const float total = block_sum(part, sh);
        // d/dx_i = (1/T) [ sum_j g_j [i = id_j] - p_i (G + gH (log p_i + H)) ]
        RowGrad g = {st.x, st.y, -a.inv_t * (total + gh * st.z), -a.inv_t * gh * LN2, n};
        float val = 0.0f;
        int32_t id = -1;
        if (threadIdx.x < n && sh.id[threadIdx.x] >= 0) {
            float sum;
            if (first_entry(sh, threadIdx.x, n, sum)) {
                id = sh.id[threadIdx.x];
                const float t = (E::get(x[id]) - st.x) * a.c - st.y;
                val = a.inv_t * sum + exp2_hw(t) * (g.a + g.b * vmax(t, T_FLOOR));
            }
        }
        __syncthreads();
        if (threadIdx.x < n) sh.id[threadIdx.x] = id, sh.val[threadIdx.x] = val;
        __syncthreads();
        write_grad<E>(g, x, out, a.C, a.c, sh);
    }
}

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
};

// The list's terms of one row, thread j < K holding entry j (K <= LG_THREADS).  Renormalised: q = softmax of the teacher's values
// over the listed classes and st describes all of the student's classes.  Bucket: q = exp(teacher), the teacher's remaining mass
// q0 = 1 - sum q against the student's mass p0 off the list, and st describes the classes OFF the list; all classes follow by
// adding the listed ones, so neither p0 nor the rest's gradient suffers the cancellation of 1 - sum p.
struct ListTerms {
    float loss;          // of the row, before weight and T^2
    float m, l2;         // all classes
    float mass;          // sum q (+ q0)
    float p0, q0;
    bool rest;           // the bucket takes part
};

template <class E>
__device__ ListTerms list_terms(const DistillArgs &a, size_t row, const typename E::raw *x, const RowStats &st, LogitsLds &sh)
{
    // sh.id / sh.val: the valid ids and their q on return
    const uint32_t j = threadIdx.x;
    int32_t id = -1;
    float t = -INFINITY, v = -INFINITY;
    if (j < a.K) {
        id = a.ids[row * a.K + j];
        if ((uint32_t)id >= a.C) id = -1;
        if (id >= 0) t = a.teacher[row * a.K + j], v = E::get(x[id]);
    }
    float q = 0.0f, logq = 0.0f;
    ListTerms r = {0.0f, st.m, st.l2, 0.0f, 0.0f, 0.0f, false};
    if (!a.bucket) {
        const float tm = block_max(t, sh);
        if (tm > -INFINITY) {
            const float e = id >= 0 ? exp2_hw((t - tm) * LOG2E) : 0.0f;
            const float tt = block_sum(e, sh);
            q = e / tt;
            logq = (t - tm) - LN2 * log2_hw(tt);
            r.mass = 1.0f;
        }
    } else {
        const double qd = id >= 0 ? exp((double)t) : 0.0;
        q = (float)qd;
        logq = t;
        const double sum = block_sum_f64(qd, sh);
        const double q0 = 1.0 - sum > 0.0 ? 1.0 - sum : 0.0;
        r.rest = st.m > -INFINITY;
        r.q0 = (float)q0;
        r.mass = (float)(r.rest ? sum + q0 : sum);
    }
    __syncthreads();
    if (j < a.K) sh.id[j] = id, sh.val[j] = q;
    __syncthreads();
    if (a.bucket) {
        float dummy;
        const bool counts = j < a.K && id >= 0 && first_entry(sh, j, a.K, dummy);
        const float top = block_max(counts ? v : -INFINITY, sh);
        const float M = vmax(st.m, top);
        if (M > -INFINITY) {
            const float rest = r.rest ? exp2_hw((st.m - M) * a.c + st.l2) : 0.0f;
            const float s = block_sum(counts ? exp2_hw((v - M) * a.c) : 0.0f, sh) + rest;
            r.m = M;
            r.l2 = log2_hw(s);
            r.p0 = rest / s;
            if (r.rest && r.q0 > 0.0f) {
                const float logp0 = (st.m - M) * a.inv_t + LN2 * (st.l2 - r.l2);
                r.loss = r.q0 * (LN2 * log2_hw(r.q0) - logp0);
            }
        } else
            r.m = M;
        if (st.m != st.m) r.m = st.m;
    }
    const float logp = (v - r.m) * a.inv_t - LN2 * r.l2;
    r.loss += block_sum(q > 0.0f || q != q ? q * (logq - logp) : 0.0f, sh);
    return r;
}

template <class E>
__device__ RowStats distill_stats(const DistillArgs &a, size_t row, const typename E::raw *x, LogitsLds &sh)
{
    if (!a.bucket) return row_stats<E>(x, a.C, a.c, sh, [](uint32_t) { return false; });
    __syncthreads();
    if (threadIdx.x < a.K) sh.id[threadIdx.x] = a.ids[row * a.K + threadIdx.x];
    __syncthreads();
    return row_stats<E>(x, a.C, a.c, sh, [&](uint32_t i) {
        for (uint32_t j = 0; j < a.K; ++j)
            if (sh.id[j] == (int32_t)i) return true;
        return false;
    });
}

template <class E>
__device__ void distill_grad(const DistillArgs &a, size_t row, const typename E::raw *x, const RowStats &st, const ListTerms &r,
                             float up, LogitsLds &sh)
{
    typename E::raw *out = (typename E::raw *)a.grad + row * a.C;
    const float coef = (a.weights ? a.weights[row] : 1.0f) * a.t * a.scale * up;
    const uint32_t j = threadIdx.x;
    int32_t id = -1;
    float val = 0.0f;
    if (j < a.K && sh.id[j] >= 0) {
        float sum;
        if (first_entry(sh, j, a.K, sum)) {
            id = sh.id[j];
            val = coef * (exp2_hw((E::get(x[id]) - r.m) * a.c - r.l2) * r.mass - sum);
        }
    }
    __syncthreads();
    if (j < a.K) sh.id[j] = id, sh.val[j] = val;
    __syncthreads();
    const float dense = a.bucket ? r.p0 * r.mass - r.q0 : r.mass;
    write_grad<E>(RowGrad{st.m, st.l2, coef * dense, 0.0f, a.K}, x, out, a.C, a.c, sh);
}

// MODE 0: losses (and statistics), 1: losses and gradient, 2: gradient from the forward call's statistics
template <class E, int MODE>
__global__ __launch_bounds__(LG_THREADS) void distill_rows_kernel(DistillArgs a)
{
    __shared__ LogitsLds sh;
    for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const typename E::raw *x = (const typename E::raw *)a.logits + row * a.stride;
        const float w = a.weights ? a.weights[row] : 1.0f;
        bool dead = w == 0.0f;                               // an ignored row: 0 whatever it holds
        RowStats st = {-INFINITY, -INFINITY, 0.0f};
        ListTerms r = {};
        if (!dead) {
            if (MODE == 2) {
                const float4 f = a.stats[row];
                st = {f.x, f.y, 0.0f};
            } else
                st = distill_stats<E>(a, row, x, sh);
            r = list_terms<E>(a, row, x, st, sh);
            dead = r.m == -INFINITY;                         // no class has any probability
        }
        if (MODE != 2 && threadIdx.x == 0) {
            a.out_rows[row] = dead ? 0.0f : w * a.t * a.t * r.loss;
            if (a.stats) a.stats[row] = make_float4(st.m, st.l2, 0.0f, 0.0f);
        }
        if (MODE != 0) {
            if (dead) {
                typename E::raw *out = (typename E::raw *)a.grad + row * a.C;
                for (uint32_t i = threadIdx.x; i < a.C; i += LG_THREADS) out[i] = E::put(0.0f);
            } else
                distill_grad<E>(a, row, x, st, r, MODE == 2 ? a.up[a.up_rows ? row : 0] : 1.0f, sh);
        }
        __syncthreads();
    }
}

// scale * sum of n floats, in double and in an order fixed by n: block b adds its run of the rows; the last launch adds the blocks.
constexpr uint32_t SUM_THREADS = 1024, SUM_RUN = 8192, SUM_BLOCKS = 512;
template <class In, class Out>
__global__ __launch_bounds__(SUM_THREADS) void sum_rows_kernel(const In *v, size_t n, size_t run, double scale, Out *out)
{
    __shared__ double part[SUM_THREADS / WAVE];
    const size_t lo = (size_t)blockIdx.x * run, hi = lo + run < n ? lo + run : n;
    double s = 0.0;
    for (size_t i = lo + threadIdx.x; i < hi; i += SUM_THREADS) s += (double)v[i];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
    if ((threadIdx.x & 63u) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t w = 1; w < SUM_THREADS / WAVE; ++w) s += part[w];
        out[blockIdx.x] = (Out)(s * scale);
    }
}
static size_t sum_run(size_t n)
{
    const size_t least = (n + SUM_BLOCKS - 1) / SUM_BLOCKS;
    return least > SUM_RUN ? least : SUM_RUN;
}

static int logits_check(const char *name, const void *logits, int dtype, size_t rows, int C, size_t stride, float temperature)
{
    if (dtype != ODBOX_DTYPE_F32 && dtype != ODBOX_DTYPE_F16 && dtype != ODBOX_DTYPE_BF16)
        return fail(ODBOX_EINVAL, "%s: dtype %d is none of ODBOX_DTYPE_*", name, dtype);
    if (C < 1 || C > ODBOX_MAX_LOGITS) return fail(ODBOX_EINVAL, "%s: C = %d is not in 1..%d", name, C, ODBOX_MAX_LOGITS);
    if (rows > (size_t)1 << 40 || stride > (size_t)1 << 40) return fail(ODBOX_EINVAL, "%s: rows or row_stride over 2^40", name);
    if (!(temperature >= 1e-6f && temperature <= 1e6f)) return fail(ODBOX_EINVAL, "%s: temperature %g is not in 1e-6..1e6", name, (double)temperature);
    if (rows && !logits) return fail(ODBOX_EINVAL, "%s: NULL logits", name);
    if ((uintptr_t)logits % (dtype == ODBOX_DTYPE_F32 ? 4 : 2)) return fail(ODBOX_EINVAL, "%s: logits are not aligned to their element", name);
    return 0;
}

static dim3 row_grid(size_t rows) { return dim3((uint32_t)(rows < 1u << 20 ? rows : 1u << 20)); }

#define LOGITS_LAUNCH(dtype, K_, ...)                                                       \
    do {                                                                                    \
        if ((dtype) == ODBOX_DTYPE_F32) { using E = F32; hipLaunchKernelGGL(K_, __VA_ARGS__); } \
        else if ((dtype) == ODBOX_DTYPE_F16) { using E = F16; hipLaunchKernelGGL(K_, __VA_ARGS__); } \
        else { using E = BF16; hipLaunchKernelGGL(K_, __VA_ARGS__); }                        \
    } while (0)

}  // namespace odbox

using namespace odbox;

extern "C" {

size_t odbox_label_logprobs_workspace(size_t rows, int C, int top_k)
{
    (void)rows, (void)C, (void)top_k;
    return 0;
}

int odbox_label_logprobs(const void *logits, int dtype, size_t rows, int C, size_t row_stride, const int32_t *labels, int top_k,
                         float temperature, float *out_logprobs, float *out_entropy, float *out_top_logprobs,
                         int32_t *out_top_labels, float *out_stats, void *workspace, size_t workspace_bytes, void *stream)
{
    const char *name = "odbox_label_logprobs";
    if (int rc = logits_check(name, logits, dtype, rows, C, row_stride, temperature)) return rc;
    if (top_k < 0 || top_k > ODBOX_MAX_TOP || top_k > C) return fail(ODBOX_EINVAL, "%s: top_k = %d is not in 0..min(C, %d)", name, top_k, ODBOX_MAX_TOP);
    if (rows == 0) return 0;
    if (out_logprobs && !labels) return fail(ODBOX_EINVAL, "%s: log-probabilities asked for, labels NULL", name);
    if (top_k && (!out_top_logprobs || !out_top_labels)) return fail(ODBOX_EINVAL, "%s: top_k = %d, NULL top output", name, top_k);
    if (!aligned16(out_stats)) return fail(ODBOX_EINVAL, "%s: out_stats must be 16-byte aligned", name);
    if (workspace_bytes < odbox_label_logprobs_workspace(rows, C, top_k)) return fail(ODBOX_ENOSPC, "%s: workspace too small", name);
    (void)workspace;
    ScoreArgs a = {logits, rows, row_stride, (uint32_t)C, (uint32_t)top_k, LOG2E / temperature, 1.0f / temperature, labels, out_logprobs, out_entropy,
                   out_top_logprobs, out_top_labels, (float4 *)out_stats};
    LOGITS_LAUNCH(dtype, score_rows_kernel<E>, row_grid(rows), dim3(LG_THREADS), 0, (hipStream_t)stream, a);
    return launch_status("label_logprobs");
}

int odbox_label_logprobs_backward(const void *logits, int dtype, size_t rows, int C, size_t row_stride, const int32_t *labels, int top_k,
                                  const int32_t *top_labels, float temperature, const float *stats, const float *upstream_logprobs,
                                  const float *upstream_entropy, const float *upstream_top, void *grad, void *stream)
{
    const char *name = "odbox_label_logprobs_backward";
    if (int rc = logits_check(name, logits, dtype, rows, C, row_stride, temperature)) return rc;
    if (top_k < 0 || top_k > ODBOX_MAX_TOP || top_k > C) return fail(ODBOX_EINVAL, "%s: top_k = %d is not in 0..min(C, %d)", name, top_k, ODBOX_MAX_TOP);
    if (rows == 0) return 0;
    if (!stats || !grad) return fail(ODBOX_EINVAL, "%s: NULL stats or grad", name);
    if (!aligned16(stats)) return fail(ODBOX_EINVAL, "%s: stats must be 16-byte aligned", name);
    if ((uintptr_t)grad % (dtype == ODBOX_DTYPE_F32 ? 4 : 2)) return fail(ODBOX_EINVAL, "%s: grad is not aligned to its element", name);
    if (upstream_logprobs && !labels) return fail(ODBOX_EINVAL, "%s: upstream_logprobs without labels", name);
    if (upstream_top && top_k && !top_labels) return fail(ODBOX_EINVAL, "%s: upstream_top without top_labels", name);
    ScoreGradArgs a = {logits, rows, row_stride, (uint32_t)C, (uint32_t)(upstream_top ? top_k : 0), LOG2E / temperature, 1.0f / temperature,
                       labels, top_labels, (const float4 *)stats, upstream_logprobs, upstream_entropy, upstream_top, grad};
    LOGITS_LAUNCH(dtype, score_grad_kernel<E>, row_grid(rows), dim3(LG_THREADS), 0, (hipStream_t)stream, a);
    return launch_status("label_logprobs_backward");
}

static int distill_check(const char *name, const void *logits, int dtype, size_t rows, int C, size_t stride, const float *teacher,
                         const int32_t *ids, int K, float temperature, int rest, const void *grad)
{
    if (int rc = logits_check(name, logits, dtype, rows, C, stride, temperature)) return rc;
    if (K < 1 || K > ODBOX_MAX_TOP) return fail(ODBOX_EINVAL, "%s: K = %d is not in 1..%d", name, K, ODBOX_MAX_TOP);
    if (rest != ODBOX_REST_RENORMALISE && rest != ODBOX_REST_BUCKET) return fail(ODBOX_EINVAL, "%s: rest = %d is none of ODBOX_REST_*", name, rest);
    if (rows && (!teacher || !ids)) return fail(ODBOX_EINVAL, "%s: NULL teacher list", name);
    if ((uintptr_t)grad % (dtype == ODBOX_DTYPE_F32 ? 4 : 2)) return fail(ODBOX_EINVAL, "%s: grad is not aligned to its element", name);
    return 0;
}

size_t odbox_distill_loss_workspace(size_t rows, int C, int K)
{
    (void)C, (void)K;
    return rows * sizeof(float) + SUM_BLOCKS * sizeof(double) + 16;
}

int odbox_distill_loss(const void *logits, int dtype, size_t rows, int C, size_t row_stride, const float *teacher_logprobs,
                       const int32_t *teacher_labels, int K, float temperature, int rest, const float *row_weights, float scale,
                       float *out_rows, float *out_loss, float *out_stats, void *grad, void *workspace, size_t workspace_bytes,
                       void *stream)
{
    const char *name = "odbox_distill_loss";
    if (int rc = distill_check(name, logits, dtype, rows, C, row_stride, teacher_logprobs, teacher_labels, K, temperature, rest, grad)) return rc;
    if (rows && !out_rows && !out_loss) return fail(ODBOX_EINVAL, "%s: NULL out_rows and out_loss", name);
    if (!aligned16(out_stats) || !aligned16(workspace)) return fail(ODBOX_EINVAL, "%s: out_stats and workspace must be 16-byte aligned", name);
    hipStream_t st = (hipStream_t)stream;
    if (rows == 0) {
        if (out_loss) {
            hipLaunchKernelGGL((sum_rows_kernel<float, float>), dim3(1), dim3(SUM_THREADS), 0, st, (const float *)nullptr, (size_t)0, (size_t)1, 0.0, out_loss);
            return launch_status("distill_loss");
        }
        return 0;
    }
    if (workspace_bytes < odbox_distill_loss_workspace(rows, C, K)) return fail(ODBOX_ENOSPC, "%s: workspace too small", name);
    if (!workspace) return fail(ODBOX_EINVAL, "%s: NULL workspace", name);
    double *partial = (double *)workspace;
    float *per_row = out_rows ? out_rows : (float *)(partial + SUM_BLOCKS);
    DistillArgs a = {logits, rows, row_stride, (uint32_t)C, (uint32_t)K, LOG2E / temperature, temperature, 1.0f / temperature, scale, rest, teacher_logprobs,
                     teacher_labels, row_weights, per_row, (float4 *)out_stats, nullptr, 0, grad};
    if (grad) LOGITS_LAUNCH(dtype, (distill_rows_kernel<E, 1>), row_grid(rows), dim3(LG_THREADS), 0, st, a);
    else LOGITS_LAUNCH(dtype, (distill_rows_kernel<E, 0>), row_grid(rows), dim3(LG_THREADS), 0, st, a);
    if (int rc = launch_status("distill_loss")) return rc;
    if (out_loss) {
        const size_t run = sum_run(rows), nb = (rows + run - 1) / run;
        if (nb == 1) {
            hipLaunchKernelGGL((sum_rows_kernel<float, float>), dim3(1), dim3(SUM_THREADS), 0, st, per_row, rows, run, (double)scale, out_loss);
        } else {
            hipLaunchKernelGGL((sum_rows_kernel<float, double>), dim3((uint32_t)nb), dim3(SUM_THREADS), 0, st, per_row, rows, run, 1.0, partial);
            hipLaunchKernelGGL((sum_rows_kernel<double, float>), dim3(1), dim3(SUM_THREADS), 0, st, partial, nb, nb, (double)scale, out_loss);
        }
        return launch_status("distill_loss sum");
    }
    return 0;
}

int odbox_distill_loss_backward(const void *logits, int dtype, size_t rows, int C, size_t row_stride, const float *teacher_logprobs,
                                const int32_t *teacher_labels, int K, float temperature, int rest, const float *row_weights, float scale,
                                const float *stats, const float *upstream, int upstream_rows, void *grad, void *stream)
{
    const char *name = "odbox_distill_loss_backward";
    if (int rc = distill_check(name, logits, dtype, rows, C, row_stride, teacher_logprobs, teacher_labels, K, temperature, rest, grad)) return rc;
    if (rows == 0) return 0;
    if (!stats || !upstream || !grad) return fail(ODBOX_EINVAL, "%s: NULL stats, upstream or grad", name);
    if (!aligned16(stats)) return fail(ODBOX_EINVAL, "%s: stats must be 16-byte aligned", name);
    DistillArgs a = {logits, rows, row_stride, (uint32_t)C, (uint32_t)K, LOG2E / temperature, temperature, 1.0f / temperature, scale, rest, teacher_logprobs,
                     teacher_labels, row_weights, nullptr, (float4 *)stats, upstream, upstream_rows, grad};
    LOGITS_LAUNCH(dtype, (distill_rows_kernel<E, 2>), row_grid(rows), dim3(LG_THREADS), 0, (hipStream_t)stream, a);
    return launch_status("distill_loss_backward");
}

}  // extern "C"
