// odbox_logits_short.hip -- class-logit operators on short rows (odbox_logits.hip has the entry points, the notation and the long rows).
#include <type_traits>

#include "odbox_logits.h"

namespace odbox {

// ------------------------------------------------------------------------------------------
// short rows: L neighbouring lanes hold a row in registers
// ------------------------------------------------------------------------------------------
// A block a row wastes itself on rows of a detector's 80 or 90 classes (392 832 of them took 4.3 ms).  Here lane l of a group of L
// keeps the S vectors l, l + L, .. of its row, so a row is read once whatever is computed from it, a sum is two (L = 4) to six
// lane exchanges, and no barrier is needed.  S is the exact number of steps, so only the last one looks at the row's end.  The last
// vector of a row that is no multiple of a vector is read (and written) back from the row's end, its first values counting as
// dropped: no access leaves the row.
constexpr int SHORT_THREADS = 256;
template <class E>
constexpr int SHORT_STEPS = E::VEC == 4 ? 6 : 4;              // 24 or 32 values a lane

template <int L>
__device__ __forceinline__ float group_max(float x)
{
    x = vmax(x, dpp_f<0xB1, 0xf>(x, x));                     // quad_perm [1,0,3,2]
    x = vmax(x, dpp_f<0x4E, 0xf>(x, x));                     // quad_perm [2,3,0,1]
    if (L >= 8) x = vmax(x, dpp_f<0x141, 0xf>(x, x));       // row_half_mirror
    if (L >= 16) x = vmax(x, dpp_f<0x140, 0xf>(x, x));       // row_mirror
    if (L >= 32) x = vmax(x, __shfl_xor(x, 16));
    if (L >= 64) x = vmax(x, __shfl_xor(x, 32));
    return x;
}
template <int L>
__device__ __forceinline__ float group_sum(float x)
{
    x += dpp_f<0xB1, 0xf>(x, x);
    x += dpp_f<0x4E, 0xf>(x, x);
    if (L >= 8) x += dpp_f<0x141, 0xf>(x, x);
    if (L >= 16) x += dpp_f<0x140, 0xf>(x, x);
    if (L >= 32) x += __shfl_xor(x, 16);
    if (L >= 64) x += __shfl_xor(x, 32);
    return x;
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u(uint32_t x) { return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xf, 0xf, false); }
template <int L, class Op>
__device__ __forceinline__ uint32_t group_fold(uint32_t x, Op op)
{
    x = op(x, dpp_u<0xB1>(x));
    x = op(x, dpp_u<0x4E>(x));
    if (L >= 8) x = op(x, dpp_u<0x141>(x));
    if (L >= 16) x = op(x, dpp_u<0x140>(x));
    if (L >= 32) x = op(x, (uint32_t)__shfl_xor(x, 16));
    if (L >= 64) x = op(x, (uint32_t)__shfl_xor(x, 32));
    return x;
}

template <class E, int L, int S>
struct ShortRow {
    static constexpr int VEC = E::VEC, PV = S * VEC;
    static constexpr bool TINY = L == 4 && S == 1;           // the only variant that meets rows shorter than a vector
    using raw = typename E::raw;
    float v[PV];
    uint32_t lane, C;

    __device__ __forceinline__ ShortRow(uint32_t classes) : lane(threadIdx.x % L), C(classes)
    {
        asm volatile("" : "+v"(lane));                       // what is computed from it is not kept from row to row
    }
    __device__ __forceinline__ bool tiny() const { return TINY && C < VEC; }
    __device__ __forceinline__ uint32_t base(int k) const
    {
        const uint32_t at = ((uint32_t)k * L + lane) * VEC;
        if (tiny()) return 0;
        return k < S - 1 || at < C - VEC ? at : C - VEC;
    }
    // leading values of the last step that belong to another vector or, past the row's end, to nobody
    __device__ __forceinline__ uint32_t drop() const { return ((S - 1) * L + lane) * VEC - base(S - 1); }
    __device__ __forceinline__ bool counts(int k, int e) const
    {
        if (tiny()) return lane == 0 && (uint32_t)e < C;
        return k < S - 1 || (uint32_t)e >= drop();
    }

    __device__ __forceinline__ void load(const raw *x)
    {
        if (!tiny()) {
            u32x4 w[S];
#pragma unroll
            for (int k = 0; k < S; ++k) w[k] = load_raw<E>(x + base(k));
#pragma unroll
            for (int k = 0; k < S; ++k) E::unpack(w[k], v + k * VEC);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = counts(0, e) ? E::get(x[e]) : -INFINITY;
        }
    }
    // f(k, e, value of v[k * VEC + e]); values that do not count are handed over as -inf
    template <class F>
    __device__ __forceinline__ void each(F f) const
    {
#pragma unroll
        for (int k = 0; k < S; ++k)
#pragma unroll
            for (int e = 0; e < VEC; ++e) f(k, e, counts(k, e) ? v[k * VEC + e] : -INFINITY);
    }
    // out[class] = f(k, e, value); a dropped value is written too, with what its own lane writes there
    template <class F>
    __device__ __forceinline__ void store(raw *out, F f) const
    {
        if (!tiny()) {
#pragma unroll
            for (int k = 0; k < S; ++k) {
                float g[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) g[e] = f(k, e, v[k * VEC + e]);
                if (k < S - 1 || drop() < VEC) store_raw<E>(out + base(k), E::pack(g));
            }
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (counts(0, e)) out[e] = E::put(f(0, e, v[e]));
        }
    }
    __device__ __forceinline__ void zero(raw *out) const { store(out, [](int, int, float) { return 0.0f; }); }
};

// Statistics of the values; a NaN comes through the sum, a row without probability has sum 0.
template <int L, bool ENT, class Each>
__device__ __forceinline__ RowStats short_stats(float c, Each each)
{
    float m = -INFINITY;
    each([&](int, int, float x) { m = vmax(m, x); });
    m = group_max<L>(m);
    const float about = m == -INFINITY ? 0.0f : m;
    float s = 0.0f, u = 0.0f;
    each([&](int, int, float x) {
        const float t = (x - about) * c, e = exp2_hw(t);
        s += e;
        if (ENT) u = __builtin_fmaf(e, vmax(t, T_FLOOR), u);
    });
    s = group_sum<L>(s);
    if (s == 0.0f) return {-INFINITY, -INFINITY, 0.0f, 0.0f};
    if (!(s < INFINITY)) return {NAN, NAN, NAN, NAN};
    const float l2 = log2_hw(s);
    return {m, l2, ENT ? LN2 * (l2 - group_sum<L>(u) / s) : 0.0f, s};
}

// 392 832 x 80 float32, five alternatives: 41 us, 3.6 TB/s, bound by the vector unit: five instructions a value and round (maximum,
// find, remove) where a 16-bit value with its class in one word needs two and a half (bfloat16: 39 us for half the bytes).
template <class E, int L, int S>
__global__ __launch_bounds__(SHORT_THREADS) void score_short_kernel(ScoreArgs a)
{
    using Row = ShortRow<E, L, S>;
    constexpr uint32_t RB = SHORT_THREADS / L;
    for (size_t row = (size_t)blockIdx.x * RB + threadIdx.x / L; row < a.rows; row += (size_t)gridDim.x * RB) {
        const typename E::raw *x = (const typename E::raw *)a.logits + row * a.stride;
        Row r(a.C);
        r.load(x);
        const RowStats st = short_stats<L, true>(a.c, [&](auto f) { r.each(f); });
        if (r.lane == 0) {
            if (a.logprobs) {
                const uint32_t lab = (uint32_t)a.labels[row];
                a.logprobs[row] = lab < a.C ? logprob_of<E>(a, st, E::get(x[lab])) : 0.0f;
            }
            if (a.entropy) a.entropy[row] = st.ent;
            if (a.stats) a.stats[row] = make_float4(st.m, st.l2, st.ent, 0.0f);
        }
        if (a.k == 0) continue;
        // One round a class: the largest value left, the lowest class that has it; 0 stands for a value that is gone.  A 16-bit value
        // and its class make one number, so that there the maximum names the class and no two are equal.
        constexpr bool PAIR = Row::VEC == 8;
        uint32_t o[Row::PV];
#pragma unroll
        for (int i = 0; i < Row::PV; ++i) {
            const int k = i / Row::VEC, e = i % Row::VEC;
            const float v = r.v[i];
            if constexpr (PAIR) o[i] = (E::order16(v) << 16) | (0xffffu - (r.base(k) + e));
            else o[i] = v != v ? 0xffffffffu : f32_ordered(v);
            if (!r.counts(k, e)) o[i] = 0;
        }
        float keep_lp = 0.0f;
        int32_t keep_id = 0;
        for (uint32_t round = 0; round < a.k; ++round) {
            uint32_t best = 0, win = 0xffffffffu;
#pragma unroll
            for (int i = 0; i < Row::PV; ++i) best = o[i] > best ? o[i] : best;
            best = group_fold<L>(best, [](uint32_t p, uint32_t q) { return p > q ? p : q; });
            float v;
            if constexpr (PAIR) {
                win = 0xffffu - (best & 0xffffu);
                v = E::value16(best >> 16);
#pragma unroll
                for (int i = 0; i < Row::PV; ++i) o[i] = o[i] == best ? 0u : o[i];
            } else {
#pragma unroll
                for (int i = Row::PV - 1; i >= 0; --i) win = o[i] == best ? r.base(i / Row::VEC) + i % Row::VEC : win;
                win = group_fold<L>(win, [](uint32_t p, uint32_t q) { return p < q ? p : q; });
#pragma unroll
                for (int i = 0; i < Row::PV; ++i) o[i] = win - r.base(i / Row::VEC) == (uint32_t)(i % Row::VEC) ? 0u : o[i];
                v = best == 0xffffffffu ? NAN : f32_unordered(best);
            }
            if (round % L == r.lane) {
                keep_id = (int32_t)win;
                keep_lp = logprob_of<E>(a, st, v);
            }
            if (round % L == L - 1 || round == a.k - 1) {    // L results at a time, side by side
                const uint32_t at = round - round % L + r.lane;
                if (at <= round) {
                    a.top_labels[row * a.k + at] = keep_id;
                    a.top_logprobs[row * a.k + at] = keep_lp;
                }
            }
        }
    }
}

// The label's and the alternatives' entries are compared with every value of a lane: two instructions a value and entry, and nothing
// to write twice.
template <class E, int L, int S>
__global__ __launch_bounds__(SHORT_THREADS) void score_grad_short_kernel(ScoreGradArgs a)
{
    using Row = ShortRow<E, L, S>;
    constexpr uint32_t RB = SHORT_THREADS / L;
    for (size_t row = (size_t)blockIdx.x * RB + threadIdx.x / L; row < a.rows; row += (size_t)gridDim.x * RB) {
        const typename E::raw *x = (const typename E::raw *)a.logits + row * a.stride;
        typename E::raw *out = (typename E::raw *)a.grad + row * a.C;
        Row r(a.C);
        r.load(x);
        const float4 st = a.stats[row];
        if (st.x == -INFINITY) {
            r.zero(out);
            continue;
        }
        auto entry = [&](uint32_t j, float &g) -> uint32_t { // class and upstream value of list entry j, the label being the last
            uint32_t id = a.C;
            g = 0.0f;
            if (j < a.k) id = (uint32_t)a.top_labels[row * a.k + j], g = a.up_top[row * a.k + j];
            else if (a.up_logprobs) id = (uint32_t)a.labels[row], g = a.up_logprobs[row];
            if (id >= a.C) id = 0xffffffffu, g = 0.0f;
            return id;
        };
        float total = 0.0f, g;
        for (uint32_t j = 0; j <= a.k; ++j) entry(j, g), total += g;
        const float gh = a.up_entropy ? a.up_entropy[row] : 0.0f;
        const float A = -a.inv_t * (total + gh * st.z), B = -a.inv_t * gh * LN2;
        float grad[Row::PV];
#pragma unroll
        for (int i = 0; i < Row::PV; ++i) {
            const float t = (r.v[i] - st.x) * a.c - st.y;
            grad[i] = exp2_hw(t) * __builtin_fmaf(B, vmax(t, T_FLOOR), A);
        }
        for (uint32_t j = 0; j <= a.k; ++j) {
            const uint32_t id = entry(j, g);
            g *= a.inv_t;
#pragma unroll
            for (int i = 0; i < Row::PV; ++i) grad[i] += id - r.base(i / Row::VEC) == (uint32_t)(i % Row::VEC) ? g : 0.0f;
        }
        r.store(out, [&](int k, int e, float) { return grad[k * Row::VEC + e]; });
    }
}

// Losses (out_rows), the gradient (GRAD) or both.  Each group has C words of LDS: -1 for a class off the list, for a listed class
// first the number of its entry (a class listed twice shows by the entries that do not find theirs), then its q.
// 392 832 x 80 float16, eight listed, by autograd: losses 25 us, gradient 38 us (130 MB, 3.4 TB/s).  24 and 43 vector instructions a value, at four
// cycles 15 and 27 us: the gradient launch computes maximum, sums and the teacher's softmax again.  (The bound on registers: 16-bit bucket
// gradients of 24 values a lane took 110 without it, so that four blocks a CU ran instead of five: 392 832 x 80 float16 64 -> 68 us.)
template <class E, int L, int S, bool BUCKET, bool GRAD>
__global__ __launch_bounds__(SHORT_THREADS, BUCKET && GRAD && E::VEC == 8 ? 8 - S : 1) void distill_short_kernel(DistillArgs a)
{
    using Row = ShortRow<E, L, S>;
    constexpr uint32_t RB = SHORT_THREADS / L;
    constexpr bool LISTED = BUCKET || GRAD;                  // the LDS is needed
    extern __shared__ __attribute__((aligned(16))) float listed[];
    const uint32_t pitch = (a.C + 3) & ~3u;
    float *list = listed + (LISTED ? (threadIdx.x / L) * pitch : 0);
    for (size_t row = (size_t)blockIdx.x * RB + threadIdx.x / L; row < a.rows; row += (size_t)gridDim.x * RB) {
        const typename E::raw *x = (const typename E::raw *)a.logits + row * a.stride;
        typename E::raw *out = (typename E::raw *)a.grad + row * a.C;
        Row r(a.C);
        const float w = a.weights ? a.weights[row] : 1.0f;
        if (w == 0.0f) {                                     // ignored: 0 whatever it holds
            if (a.out_rows && r.lane == 0) {
                a.out_rows[row] = 0.0f;
                if (a.stats) a.stats[row] = make_float4(-INFINITY, -INFINITY, 0.0f, 0.0f);
            }
            if (GRAD) r.zero(out);
            continue;
        }
        r.load(x);
        const float *teacher = a.teacher + row * a.K;
        const int32_t *ids = a.ids + row * a.K;
        auto entry = [&](uint32_t j, float &t) -> uint32_t {
            const uint32_t id = (uint32_t)ids[j];
            t = id < a.C ? teacher[j] : -INFINITY;
            return id;
        };
        auto fence = [] { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); };    // one wave's LDS accesses stay in order

        uint32_t own = 0;                                    // bit i: this lane's i-th entry is its class's first or only one
        bool twice = false;
        if (LISTED) {
            fence();
            for (uint32_t i = r.lane * 4; i < pitch; i += L * 4) *(float4 *)(list + i) = make_float4(-1.0f, -1.0f, -1.0f, -1.0f);
            fence();
            for (uint32_t j = r.lane; j < a.K; j += L)
                if ((uint32_t)ids[j] < a.C) list[ids[j]] = (float)j;
            fence();
            for (uint32_t j = r.lane, i = 0; j < a.K; j += L, ++i) {
                if ((uint32_t)ids[j] >= a.C) continue;
                if (list[ids[j]] == (float)j) own |= 1u << i;
                else twice = true;
            }
            fence();
            twice = group_fold<L>(twice ? 1u : 0u, [](uint32_t p, uint32_t q) { return p | q; }) != 0;
        }
        auto off_list = [&](int k, int e) { return list[r.base(k) + e] < 0.0f; };
        RowStats st;
        if (BUCKET) {
            uint32_t bits = 0;                               // the values off the list
            r.each([&](int k, int e, float) { bits |= (r.counts(k, e) && off_list(k, e) ? 1u : 0u) << (k * Row::VEC + e); });
            st = short_stats<L, false>(a.c, [&](auto f) { r.each([&](int k, int e, float v) { f(k, e, bits >> (k * Row::VEC + e) & 1u ? v : -INFINITY); }); });
        } else
            st = short_stats<L, false>(a.c, [&](auto f) { r.each(f); });

        // the list's terms, as in list_terms()
        float about = 0.0f, tt = 0.0f, mass = 0.0f, q0 = 0.0f, loss = 0.0f;
        float m = st.m, l2 = st.l2, dense = 0.0f, t;
        bool rest = false;
        if (!BUCKET) {
            float tm = -INFINITY;
            for (uint32_t j = r.lane; j < a.K; j += L) entry(j, t), tm = vmax(tm, t);
            tm = group_max<L>(tm);
            if (tm > -INFINITY) about = tm;
            for (uint32_t j = r.lane; j < a.K; j += L) entry(j, t), tt += exp2_hw((t - about) * LOG2E);
            tt = group_sum<L>(tt);
            mass = tt == 0.0f ? 0.0f : tt == tt ? 1.0f : NAN;    // the maximum does not see a NaN, the sum does
        } else {
            double sum = 0.0;
            for (uint32_t j = r.lane; j < a.K; j += L) entry(j, t), sum += exp_wide(t);
#pragma unroll
            for (int off = 1; off < L; off <<= 1) sum += __shfl_xor(sum, off);
            const double left = 1.0 - sum;
            rest = st.m > -INFINITY;
            q0 = left > 0.0 ? (float)left : left != left ? NAN : 0.0f;
            mass = rest ? (float)sum + q0 : (float)sum;
            float top = -INFINITY;
            for (uint32_t j = r.lane, i = 0; j < a.K; j += L, ++i)
                if (own >> i & 1u) top = vmax(top, E::get(x[ids[j]]));
            top = group_max<L>(top);
            m = vmax(st.m, top);
            const float to = m > -INFINITY ? m : 0.0f;
            float on = 0.0f;
            for (uint32_t j = r.lane, i = 0; j < a.K; j += L, ++i)
                if (own >> i & 1u) on += exp2_hw((E::get(x[ids[j]]) - to) * a.c);
            on = group_sum<L>(on);
            if (m > -INFINITY) {
                const float off = rest ? st.s * exp2_hw((st.m - m) * a.c) : 0.0f;
                l2 = log2_hw(on + off);
                const BucketTerms b = bucket_terms(on, off, (float)sum, q0, (st.m - m) * a.inv_t + LN2 * (st.l2 - l2));
                dense = b.dense;
                if (rest) loss = b.rest;
            }
            if (st.m != st.m || on != on) m = NAN;           // (the maxima do not see a NaN)
        }
        auto q_of = [&](float v) { return BUCKET ? exp_split(v) : tt != 0.0f ? exp2_hw((v - about) * LOG2E) / tt : 0.0f; };
        float terms = 0.0f;
        for (uint32_t j = r.lane, i = 0; j < a.K; j += L, ++i) {
            const uint32_t id = entry(j, t);
            if (id >= a.C) continue;
            const float q = q_of(t);
            if (a.out_rows && (q > 0.0f || q != q)) {
                const float logq = BUCKET ? t : (t - about) - LN2 * log2_hw(tt);
                terms += q * (logq - ((E::get(x[id]) - m) * a.inv_t - LN2 * l2));
            }
            if (GRAD && (own >> i & 1u)) {
                float sum = q;
                if (twice) {
                    sum = 0.0f;
                    for (uint32_t n = 0; n < a.K; ++n)
                        if ((uint32_t)ids[n] == id) sum += q_of(teacher[n]);
                }
                list[id] = sum;
            }
        }
        if (mass != mass && m > -INFINITY) m = mass;         // a NaN or +inf among the teacher's values, except for an empty row
        if (m != m) loss = m;                                // also where nothing is listed
        const bool dead = m == -INFINITY;
        if (a.out_rows) {
            loss += group_sum<L>(terms);
            if (r.lane == 0) {
                a.out_rows[row] = dead ? 0.0f : w * a.t * a.t * loss;
                if (a.stats) a.stats[row] = make_float4(st.m, st.l2, st.s, 0.0f);
            }
        }
        if (GRAD) {
            fence();
            if (dead) {
                r.zero(out);
            } else {
                const float coef = w * a.t * a.scale * (a.up ? a.up[a.up_rows ? row : 0] : 1.0f);
                const float none = m != m ? m : 0.0f;        // off the list where nothing there has a probability
                r.store(out, [&](int k, int e, float v) {
                    const float b = list[r.base(k) + e];
                    if (!BUCKET) return coef * (exp2_hw((v - st.m) * a.c - st.l2) * mass - (b < 0.0f ? 0.0f : b));
                    const bool on = b >= 0.0f || b != b;
                    const float p = exp2_hw((v - (on ? m : st.m)) * a.c - (on ? l2 : st.l2));
                    return on ? coef * (p * mass - b) : rest ? coef * dense * p : none;
                });
            }
            fence();
        }
    }
}

// A short row of nv vectors goes to the smallest group of 4, 8, .. 64 lanes that holds it in SHORT_STEPS steps.
int short_limit(int dtype) { return dtype == ODBOX_DTYPE_F32 ? 64 * SHORT_STEPS<F32> * 4 : 64 * SHORT_STEPS<F16> * 8; }
static dim3 short_grid(size_t rows, int L)
{
    const size_t per = SHORT_THREADS / L;
    return work_grid((rows + per - 1) / per);
}
template <int V>
using Constant = std::integral_constant<int, V>;
template <class E, int L, int S, class F>
static void short_lanes(int nv, F f)
{
    if (nv > L * SHORT_STEPS<E>) {
        if constexpr (L < 64) short_lanes<E, 2 * L, SHORT_STEPS<E> / 2 + 1>(nv, f);
    } else if (nv > L * S) {
        if constexpr (S < SHORT_STEPS<E>) short_lanes<E, L, S + 1>(nv, f);
    } else
        f(E(), Constant<L>(), Constant<S>());
}
template <class F>
static void short_variant(int dtype, int C, F f)
{
    if (dtype == ODBOX_DTYPE_F32) short_lanes<F32, 4, 1>((C + 3) / 4, f);
    else if (dtype == ODBOX_DTYPE_F16) short_lanes<F16, 4, 1>((C + 7) / 8, f);
    else short_lanes<BF16, 4, 1>((C + 7) / 8, f);
}
// The short kernel's selection costs a round for every class on L lanes, the wave's threshold about the same for any k.  Measured
// (float32, rounds / threshold): 100 000 x 300, k 32 (16 lanes) 162 / 281 us; 40 000 x 600, k 16 (32 lanes) 77 / 97;
// 20 000 x 1000, k 10 (64 lanes) 49 / 55; 20 000 x 1400, k 20 (64 lanes) 110 / 62.
bool score_is_short(int dtype, int C, int k)
{
    if (C > short_limit(dtype)) return false;
    int lanes = 64;
    short_variant(dtype, C, [&](auto, auto l, auto) { lanes = decltype(l)::value; });
    return lanes == 4 || k * lanes <= 640;
}

void score_short(int dtype, const ScoreArgs &a, hipStream_t st)
{
    short_variant(dtype, (int)a.C, [&](auto e, auto l, auto n) {
        using E = decltype(e);
        constexpr int L = decltype(l)::value, S = decltype(n)::value;
        hipLaunchKernelGGL((score_short_kernel<E, L, S>), short_grid(a.rows, L), dim3(SHORT_THREADS), 0, st, a);
    });
}

void score_grad_short(int dtype, const ScoreGradArgs &a, hipStream_t st)
{
    short_variant(dtype, (int)a.C, [&](auto e, auto l, auto n) {
        using E = decltype(e);
        constexpr int L = decltype(l)::value, S = decltype(n)::value;
        hipLaunchKernelGGL((score_grad_short_kernel<E, L, S>), short_grid(a.rows, L), dim3(SHORT_THREADS), 0, st, a);
    });
}

void distill_short(int dtype, int rest, bool grad, const DistillArgs &a, hipStream_t st)
{
    const size_t rows = a.rows;
    short_variant(dtype, (int)a.C, [&](auto e, auto l, auto n) {
        using E = decltype(e);
        constexpr int L = decltype(l)::value, S = decltype(n)::value;
        const size_t lds = (size_t)(SHORT_THREADS / L) * ((a.C + 3) & ~3u) * sizeof(float);
        const dim3 grid = short_grid(rows, L), block(SHORT_THREADS);
        if (rest == ODBOX_REST_BUCKET) {
            if (grad) hipLaunchKernelGGL((distill_short_kernel<E, L, S, true, true>), grid, block, lds, st, a);
            else hipLaunchKernelGGL((distill_short_kernel<E, L, S, true, false>), grid, block, lds, st, a);
        } else {
            if (grad) hipLaunchKernelGGL((distill_short_kernel<E, L, S, false, true>), grid, block, lds, st, a);
            else hipLaunchKernelGGL((distill_short_kernel<E, L, S, false, false>), grid, block, 0, st, a);
        }
    });
}

}  // namespace odbox
