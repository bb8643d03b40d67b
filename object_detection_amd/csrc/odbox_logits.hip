// odbox_logits.hip -- operators on rows of class logits: log-probabilities of given labels with entropy and top
// alternatives, and distillation from a teacher's top classes, forward and backward.  No counterpart in the reference,
// whose only softmax is metric.py:19-20; the entry points stand beside odbox_focal_loss_rows.
//
// Notation of every kernel here: a row x of C logits, c = log2(e) / temperature, m = the row's largest logit,
// s = sum 2^((x - m) c), l2 = log2(s); log2 p_i = (x_i - m) c - l2.  m is taken out BEFORE the multiplication, so that rows
// of large or shifted logits lose nothing; log-probabilities that are returned are (x_i - m) / T - ln2 l2, which stays finite as
// far as float32 reaches.  Sums, maxima and outputs other than gradients are 32-bit floats.
#include <type_traits>

#include "odbox_logits.h"

namespace odbox {

constexpr uint32_t TOP_CAP = 1024;               // candidates of a row's top classes
constexpr uint32_t MAX_WAVES = 16;
constexpr uint32_t LIST_MAX = ODBOX_MAX_TOP + 1;

// What one block shares.
struct LogitsLds {
    float f[MAX_WAVES];
    float3 part[MAX_WAVES];
    uint32_t count;
    uint32_t pick[2];
    alignas(16) int32_t id[LIST_MAX + 3];        // listed classes; -1: none, or listed before
    float val[LIST_MAX];                         // of a listed class: its upstream value, or its q over all its entries
    float q[ODBOX_MAX_TOP], logq[ODBOX_MAX_TOP], x[ODBOX_MAX_TOP];   // of a teacher's entry, and the student's logit there
    float sum[4];
};
struct TopLds {
    alignas(16) uint32_t group[256];             // group maxima of the selection; the radix histogram
    uint64_t key[TOP_CAP];                       // candidates; while they are collected, TOP_CAP / waves to each wave
};

template <int NT, class Op>
__device__ __forceinline__ float block_reduce(float v, float none, LogitsLds &sh, Op op)
{
    v = wave_reduce(v, none, op);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) sh.f[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh.f[0];
#pragma unroll
    for (int w = 1; w < NT / WAVE; ++w) v = op(v, sh.f[w]);
    return v;
}
template <int NT>
__device__ __forceinline__ float block_max(float v, LogitsLds &sh) { return block_reduce<NT>(v, -INFINITY, sh, [](float a, float b) { return vmax(a, b); }); }
template <int NT>
__device__ __forceinline__ float block_sum(float v, LogitsLds &sh) { return block_reduce<NT>(v, 0.0f, sh, [](float a, float b) { return a + b; }); }

// ------------------------------------------------------------------------------------------
// softmax statistics of a row
// ------------------------------------------------------------------------------------------
// One thread's share of a row in one pass: maximum m, s = sum 2^(x c - mc) and u = sum 2^(x c - mc) (x c - mc), mc = m c as
// rounded (nmc = -mc).  The fused multiply-add rounds x c - mc once, and join() takes the rounding of mc out again.
struct Running {
    float m, nmc, s, u;
};
__device__ __forceinline__ Running running_start(float c) { return {M_START, -(M_START * c), 0.0f, 0.0f}; }

// N values at once: one maximum, one rescaling.  A class at -inf adds 0; what a NaN, an infinity or values whose product with c
// overflows do to s, row_ok() sees.
template <int N, bool ENT>
__device__ __forceinline__ void absorb(const float *v, float c, Running &r)
{
    float g = r.m;
    if (N == 1) g = vmax(g, v[0]);
#pragma unroll
    for (int i = 0; i + 1 < N; i += 2) g = vmax3(g, v[i], v[i + 1]);
    const float nmc = -(g * c), d = nmc - r.nmc, f = exp2_hw(d);
    if (ENT) r.u = __builtin_fmaf(d, r.s, r.u) * f;
    r.s *= f;
    r.m = g;
    r.nmc = nmc;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float t = __builtin_fmaf(v[i], c, nmc), e = exp2_hw(t);
        s += e;
        if (ENT) r.u = __builtin_fmaf(e, vmax(t, T_FLOOR), r.u);
    }
    r.s += s;
}

// Shares of a wave, then of a block, about the common maximum M: x -> float3(M, sum 2^((x - M) c), sum of the same times its exponent)
__device__ __forceinline__ float3 wave_join(const Running &r, float c)
{
    const float M = wave_max(r.m);
    const float D = (r.m - M) * c + __builtin_fmaf(-r.m, c, -r.nmc), f = exp2_hw(D);
    const bool some = r.s != 0.0f;               // (a share without classes would make 0 * inf out of its M_START)
    return make_float3(M, wave_sum(some ? r.s * f : 0.0f), wave_sum(some ? __builtin_fmaf(D, r.s, r.u) * f : 0.0f));
}
__device__ __forceinline__ float3 join(const float3 *part, uint32_t n, float c)
{
    float M = part[0].x;
    for (uint32_t w = 1; w < n; ++w) M = vmax(M, part[w].x);
    float s = 0.0f, u = 0.0f;
    for (uint32_t w = 0; w < n; ++w) {
        const float3 p = part[w];
        const float D = (p.x - M) * c, f = exp2_hw(D);
        if (p.y != 0.0f) s += p.y * f, u += __builtin_fmaf(D, p.y, p.z) * f;
    }
    return make_float3(M, s, u);
}
template <int NT>
__device__ __forceinline__ float3 block_join(const Running &r, float c, LogitsLds &sh)
{
    const float3 p = wave_join(r, c);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) sh.part[threadIdx.x >> 6] = p;
    __syncthreads();
    return join(sh.part, NT / WAVE, c);
}
// Whether one pass sufficed.  Not so where no class lies above M_START (all forbidden, all at the type's lowest value) or
// where a NaN, an infinity or an overflow of m c made the sum 0, infinite or NaN.
__device__ __forceinline__ bool row_ok(const float3 &j) { return j.y > 0.0f && j.y < INFINITY; }
__device__ __forceinline__ RowStats stats_of(const float3 &j)
{
    const float l2 = log2_hw(j.y);
    return {j.x, l2, LN2 * (l2 - j.z / j.y), j.y};
}

// Two passes over the row by the whole block, for the rows that are not row_ok; the classes among the K of sh.id are left out.
// (A call, so that it costs the kernels no registers.)
template <class E, int NT>
__device__ __attribute__((noinline)) RowStats careful_stats(const typename E::raw *x, uint32_t C, float c, uint32_t K, LogitsLds &sh)
{
    auto skip = [&](uint32_t i) {
        for (uint32_t j = 0; j < K; ++j)
            if (sh.id[j] == (int32_t)i) return true;
        return false;
    };
    float m = -INFINITY, bad = 0.0f;
    for (uint32_t i = threadIdx.x; i < C; i += NT) {
        const float v = E::get(x[i]);
        if (skip(i)) continue;
        if (v != v || v == INFINITY) bad = 1.0f;
        m = vmax(m, v);
    }
    m = block_max<NT>(m, sh);
    bad = block_max<NT>(bad, sh);
    if (bad != 0.0f) return {NAN, NAN, NAN, NAN};
    if (m == -INFINITY) return {m, -INFINITY, 0.0f, 0.0f};
    float s = 0.0f, u = 0.0f;
    for (uint32_t i = threadIdx.x; i < C; i += NT) {
        if (skip(i)) continue;
        const float t = (E::get(x[i]) - m) * c, e = exp2_hw(t);
        s += e;
        u += e * vmax(t, T_FLOOR);
    }
    s = block_sum<NT>(s, sh);
    u = block_sum<NT>(u, sh);
    const float l2 = log2_hw(s);
    return {m, l2, LN2 * (l2 - u / s), s};
}

// n classes of a row as seen by 16-byte loads: `head` classes up to the first boundary, nvec vectors, the rest.  Head and rest, fewer than
// two vectors together, are the span's edge: class `edge(t)` belongs to thread t.  (Vectors across the boundaries read 25 % slower.)
template <class E>
struct Span {
    uint32_t n, head, nvec, edges;
    __device__ __forceinline__ Span(const typename E::raw *x, uint32_t count) : n(count)
    {
        const uint32_t gap = (uint32_t)((0u - (uint32_t)(uintptr_t)x) & 15u) / (uint32_t)sizeof(typename E::raw);
        head = gap < n ? gap : n;
        nvec = (n - head) / E::VEC;
        edges = n - nvec * E::VEC;
    }
    __device__ __forceinline__ uint32_t edge(uint32_t t) const { return t < head ? t : t + nvec * E::VEC; }
};

// Which of a span's classes are left out: a word for every 32 values that a thread takes in one go (bit j for value j), the edge's last.
// word(i): that of vector i (NT threads take the vectors in turn), bit(i): of its first value.
template <class E, int NT>
struct Mask {
    static constexpr uint32_t VEC = E::VEC, U = 32 / E::VEC;
    static __device__ __forceinline__ uint32_t words(uint32_t nvec) { return (nvec + U * NT - 1) / (U * NT) * NT + 1; }
    static __device__ __forceinline__ uint32_t word(uint32_t i) { return i / (U * NT) * NT + i % NT; }
    static __device__ __forceinline__ uint32_t bit(uint32_t i) { return i / NT % U * VEC; }
};

// A block's pass over a span.
template <class E, int NT, bool ENT, bool MASK, bool PASSING>
__device__ __forceinline__ Running scan_classes(const typename E::raw *x, const Span<E> &span, float c, const uint32_t *mask)
{
    constexpr int VEC = E::VEC, U = 32 / VEC;
    using M = Mask<E, NT>;
    const uint32_t nvec = span.nvec;
    const typename E::raw *body = x + span.head;
    Running r = running_start(c);
    uint32_t i = threadIdx.x;
    for (; i + (U - 1) * NT < nvec; i += U * NT) {
        u32x4 w[U];
#pragma unroll
        for (int k = 0; k < U; ++k) w[k] = load_raw<E, PASSING>(body + (size_t)(i + k * NT) * VEC);
        float v[U * VEC];
#pragma unroll
        for (int k = 0; k < U; ++k) E::unpack(w[k], v + k * VEC);
        if (MASK) {
            const uint32_t b = mask[M::word(i)];
            if (__any(b)) {
#pragma unroll
                for (int j = 0; j < U * VEC; ++j) v[j] = b >> j & 1u ? -INFINITY : v[j];
            }
        }
        absorb<U * VEC, ENT>(v, c, r);
    }
    for (; i < nvec; i += NT) {
        float v[VEC];
        E::unpack(load_raw<E, PASSING>(body + (size_t)i * VEC), v);
        if (MASK) {
            const uint32_t b = mask[M::word(i)] >> M::bit(i);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = b >> e & 1u ? -INFINITY : v[e];
        }
        absorb<VEC, ENT>(v, c, r);
    }
    if (threadIdx.x < span.edges) {
        float v = E::get(x[span.edge(threadIdx.x)]);
        if (MASK) v = mask[M::words(nvec) - 1] >> threadIdx.x & 1u ? -INFINITY : v;
        absorb<1, ENT>(&v, c, r);
    }
    return r;
}

// ------------------------------------------------------------------------------------------
// top classes
// ------------------------------------------------------------------------------------------
// Order of the top alternatives: value descending, then index ascending; NaN above everything.  56 significant bits.
__device__ __forceinline__ uint64_t top_key(float v, uint32_t i)
{
    const uint32_t o = v != v ? 0xffffffffu : f32_ordered(v);
    return ((uint64_t)o << 24) | (0xffffffu - i);
}
__device__ __forceinline__ uint32_t top_index(uint64_t k) { return 0xffffffu - ((uint32_t)k & 0xffffffu); }
__device__ __forceinline__ float top_value(uint64_t k)
{
    const uint32_t o = (uint32_t)(k >> 24);
    return o == 0xffffffffu ? NAN : f32_unordered(o);
}

// n candidates in top.key, unordered, the k largest of the whole among them: each counts the larger ones, out(rank, key) is
// called for the first k.  Where there are more threads than candidates, 2^sh lanes share one.
template <int NT, class Out>
__device__ __forceinline__ void rank_candidates(uint32_t n, uint32_t k, const TopLds &top, Out out)
{
    uint32_t sh = 0;
    while (sh < 6 && (n << (sh + 1)) <= NT) ++sh;
    const uint32_t lanes = 1u << sh, sub = threadIdx.x & (lanes - 1), step = NT >> sh;
    for (uint32_t t0 = 0; t0 < n; t0 += 2 * step) {
        const uint32_t t = t0 + (threadIdx.x >> sh), t2 = t + step;
        const uint64_t mine = top.key[t < n ? t : 0], mine2 = top.key[t2 < n ? t2 : 0];
        uint32_t rank = 0, rank2 = 0, j = sub;
        for (; j + 7 * lanes < n; j += 8 * lanes) {
            uint64_t q[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = top.key[j + i * lanes];
#pragma unroll
            for (int i = 0; i < 8; ++i) rank += q[i] > mine, rank2 += q[i] > mine2;
        }
        for (; j < n; j += lanes) rank += top.key[j] > mine, rank2 += top.key[j] > mine2;
        for (uint32_t off = 1; off < lanes; off <<= 1) rank += __shfl_xor(rank, off), rank2 += __shfl_xor(rank2, off);
        if (t < n && sub == 0 && rank < k) out(rank, mine);
        if (t2 < n && sub == 0 && rank2 < k) out(rank2, mine2);
    }
}

// The k (<= ODBOX_MAX_TOP, <= n) largest of n unique keys: the k-th key by a radix selection of eight bits a pass, then exactly k
// keys are collected.  Right for every input, eight passes: where the threshold below keeps too few or too many candidates.  That is also where a mask
// leaves fewer than k classes of a row or segment, and it is slow: 4096 x 32768 bfloat16, 64 classes, 78 us with 99 % forbidden, 3 ms with
// 99.9 %; 48 x 65537 float32, 20 classes, 20 and 139 us.
// They end up in top.key in order.  (A call: key is a plain object.)
template <int NT, class Key>
__device__ __attribute__((noinline)) void top_radix(uint32_t n, uint32_t k, LogitsLds &sh, TopLds &top, Key key)
{
    uint64_t prefix = 0;
    uint32_t want = k;
    for (int shift = 48; shift >= 0; shift -= 8) {
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < 256; i += NT) top.group[i] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < n; i += NT) {
            const uint64_t q = key(i);
            if ((q >> shift >> 8) == prefix) atomicAdd(&top.group[(uint32_t)(q >> shift) & 255u], 1u);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            uint32_t above = 0, b = 255;
            while (b > 0 && above + top.group[b] < want) above += top.group[b--];
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
    for (uint32_t i = threadIdx.x; i < n; i += NT) {
        const uint64_t q = key(i);
        if (q >= prefix) top.key[atomicAdd(&sh.count, 1u)] = q;       // unique keys: exactly k of them
    }
    __syncthreads();
    uint64_t mine[(ODBOX_MAX_TOP + NT - 1) / NT];
    uint32_t rank[(ODBOX_MAX_TOP + NT - 1) / NT];
#pragma unroll
    for (uint32_t h = 0; h < (ODBOX_MAX_TOP + NT - 1) / NT; ++h) {
        const uint32_t t = threadIdx.x + h * NT;
        mine[h] = t < k ? top.key[t] : 0;
        rank[h] = 0;
        for (uint32_t j = 0; j < k; ++j) rank[h] += top.key[j] > mine[h];
    }
    __syncthreads();
#pragma unroll
    for (uint32_t h = 0; h < (ODBOX_MAX_TOP + NT - 1) / NT; ++h)
        if (threadIdx.x + h * NT < k) top.key[rank[h]] = mine[h];
    __syncthreads();
}
template <class E>
struct ClassKey {
    const typename E::raw *x;
    uint32_t first;
    __device__ __forceinline__ uint64_t operator()(uint32_t i) const { return top_key(E::get(x[i]), first + i); }
};
struct StoredKey {
    const uint64_t *keys;
    __device__ __forceinline__ uint64_t operator()(uint32_t i) const { return keys[i]; }
};

// Groups of the threshold: at least 2 k of them keep about 1.4 k candidates of values in no particular order.
__device__ __forceinline__ uint32_t top_groups(uint32_t k) { return k <= 32 ? 64 : k <= 64 ? 128 : 256; }

// A value (in f32_ordered form) that at least k of the row's classes reach and few more do: the k-th largest of G group maxima in
// top.group, its last 12 bits cleared.  One wave finds it bit by bit, counting by ballots: 20 steps of some 60 cycles, where letting
// every group count the larger ones takes four times as long at 256 groups.
template <int NT>
__device__ __forceinline__ uint32_t top_threshold(uint32_t G, uint32_t k, LogitsLds &sh, TopLds &top)
{
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    if (threadIdx.x < WAVE) {
        uint32_t g[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) g[i] = (uint32_t)i * 64 < G ? top.group[i * 64 + threadIdx.x] : 0u;
        uint32_t tau = 0;
        for (uint32_t bit = 1u << 31; bit >= 1u << 12; bit >>= 1) {
            const uint32_t t = tau | bit;
            uint32_t n = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) n += __popcll(__ballot(g[i] >= t));
            if (n >= k) tau = t;
        }
        if (threadIdx.x == 0) sh.pick[0] = tau;
    }
    __syncthreads();
    return sh.pick[0];
}
__device__ __forceinline__ void push_candidate(uint64_t key, LogitsLds &sh, TopLds &top)
{
    const uint32_t at = atomicAdd(&sh.count, 1u);
    if (at < TOP_CAP) top.key[at] = key;
}

// A row, or a segment of one, in the registers of NT threads: vector i of its span at thread i % NT, one class of the edge at each of
// the first threads.  What is read twice (the top classes, a gradient) is read from memory once.
template <class E, int NT>
struct Resident {
    static constexpr int R = 16, VEC = E::VEC, N = 16, STEP = N / VEC;       // N values at a time
    using raw = typename E::raw;
    u32x4 w[R];
    float edge;
    uint32_t tid;

    template <bool PASSING>
    __device__ __forceinline__ void load(const raw *x, const Span<E> &span)
    {
        const raw *body = x + span.head;
        forget_thread();
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const uint32_t i = k * NT + tid;
            w[k] = E::none();
            if (i < span.nvec) w[k] = load_raw<E, PASSING>(body + (size_t)i * VEC);
        }
        edge = tid < span.edges ? E::get(x[span.edge(tid)]) : -INFINITY;
    }
    // The thread's number as something new: what is computed from it (an index for every value) is not kept from row to row.
    __device__ __forceinline__ void forget_thread()
    {
        tid = threadIdx.x;
        asm volatile("" : "+v"(tid));
    }
    // Keeps the compiler from holding the unpacked values (two to one register) between two uses of the row.
    __device__ __forceinline__ void forget()
    {
        forget_thread();
#pragma unroll
        for (int k = 0; k < R; ++k) asm volatile("" : "+v"(w[k]));
    }
    // f(k, v): N values from vector k on, for the steps that hold any
    template <class F>
    __device__ __forceinline__ void each(const Span<E> &span, F f) const
    {
#pragma unroll
        for (int k = 0; k < R; k += STEP) {
            if ((uint32_t)k * NT < span.nvec) {
                float v[N];
#pragma unroll
                for (int j = 0; j < STEP; ++j) E::unpack(w[k + j], v + j * VEC);
                f(k, v);
            }
        }
    }
};

// The k best of the classes in r, whose indices start at first; m: the thread's largest value.  free_registers() is called when r is
// no longer needed, and may load the next row into it.
template <class E, int NT, class Free, class Out>
__device__ __forceinline__ void top_classes(Resident<E, NT> &r, const typename E::raw *x, const Span<E> &span, uint32_t first, uint32_t k, float m,
                                            bool ok, LogitsLds &sh, TopLds &top, Free free_registers, Out out)
{
    using Row = Resident<E, NT>;
    constexpr int VEC = E::VEC, WAVES = NT / WAVE;
    const uint32_t n = span.n;
    constexpr uint32_t ROOM = TOP_CAP / WAVES;
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63u;
    bool few = false;
    uint32_t have = 0;
    if (ok) {
        // group maxima: of neighbouring threads, or of parts of a thread's values where there are too few threads
        const uint32_t G = top_groups(k);
        __syncthreads();
        if (NT >= 256 || G == 64) {
            const uint32_t lanes = NT / G;
            uint32_t v = f32_ordered(m);
            for (uint32_t off = 1; off < lanes; off <<= 1) {
                const uint32_t o = __shfl_xor(v, off);
                v = o > v ? o : v;
            }
            if (threadIdx.x % lanes == 0) top.group[threadIdx.x / lanes] = v;
        } else {
            // a single wave and k > 32: the values of a thread fall into four groups, or into two
            float g[4] = {r.edge, M_START, M_START, M_START};
            r.each(span, [&](int kk, const float *v) {
#pragma unroll
                for (int j = 0; j < Resident<E, NT>::N; ++j) g[(kk + j / VEC) & 3] = vmax(g[(kk + j / VEC) & 3], v[j]);
            });
            if (G == 128) g[0] = vmax(g[0], g[2]), g[1] = vmax(g[1], g[3]);
            for (uint32_t part = 0; part < G / 64; ++part)
                top.group[part * 64 + threadIdx.x] = f32_ordered(vmax(part == 0 ? g[0] : part == 1 ? g[1] : part == 2 ? g[2] : g[3], M_START));
        }
        const float tau = f32_unordered(top_threshold<NT>(G, k, sh, top));
        // Candidates by wave: a ballot per value, so positions need no atomics and their order no luck.  A miss costs two
        // instructions; what a hit stores (value and index, made a key later) is kept short, some 22 of a wave's 8192 values hit.
        const uint32_t mine = span.head + r.tid * VEC;
        uint2 *list = (uint2 *)top.key + wave * ROOM;
        auto look = [&](float v, uint32_t at) {
            const uint64_t hit = __ballot(v >= tau);
            if (hit == 0) return;
            const uint32_t pos = have + __builtin_amdgcn_mbcnt_hi((uint32_t)(hit >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hit, 0u));
            if (v >= tau && pos < ROOM) list[pos] = make_uint2(__float_as_uint(v), at);
            have += __popcll(hit);
        };
        if (__any(m >= tau)) {
            r.each(span, [&](int kk, const float *v) {
#pragma unroll
                for (int j = 0; j < Row::N; ++j) look(v[j], mine + (kk + j / VEC) * NT * VEC + j % VEC);
            });
            look(r.edge, span.edge(r.tid));
        }
    }
    free_registers();
    if (ok) {
        // the waves' lists side by side (places beyond the span hold -inf, tau is M_START or more: they never count)
        const bool over = have > ROOM;
        const uint2 *list = (const uint2 *)top.key + wave * ROOM;
        uint64_t key[(ROOM + 63) / 64 < 4 ? (ROOM + 63) / 64 : 4];       // (a single wave's list may be longer: in place, piece by piece)
        constexpr uint32_t PIECE = sizeof(key) / 8 * 64;
        auto read = [&](uint32_t from) {
#pragma unroll
            for (uint32_t i = 0; i < PIECE / 64; ++i) {
                const uint32_t t = from + i * 64 + lane;
                if (t < have) key[i] = top_key(__uint_as_float(list[t].x), first + list[t].y);
            }
        };
        auto write = [&](uint32_t from, uint32_t to) {
#pragma unroll
            for (uint32_t i = 0; i < PIECE / 64; ++i) {
                const uint32_t t = i * 64 + lane;
                if (from + t < have) top.key[to + t] = key[i];
            }
        };
        if (WAVES > 1) {
            static_assert(WAVES == 1 || PIECE >= ROOM, "a wave's list fits one piece");
            if (!over) read(0);
            if (lane == 0) sh.f[wave] = over ? 1e9f : (float)have;
            __syncthreads();
            uint32_t base = 0, all = 0;
            for (int i = 0; i < WAVES; ++i) {
                const uint32_t c = sh.f[i] > 1e8f ? 2 * TOP_CAP : (uint32_t)sh.f[i];
                if ((uint32_t)i < wave) base += c;
                all += c;
            }
            few = all >= k && all <= TOP_CAP;
            if (few) write(0, base);
            have = all;
        } else {
            few = have >= k && !over;
            if (few)
                for (uint32_t from = 0; from < have; from += PIECE) read(from), write(from, from);
        }
        __syncthreads();
        if (few) rank_candidates<NT>(have, k, top, out);
        __syncthreads();
    }
    if (!few) {
        top_radix<NT>(n, k, sh, top, ClassKey<E>{x, first});
        for (uint32_t t = threadIdx.x; t < k; t += NT) out(t, top.key[t]);
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------
// scores
// ------------------------------------------------------------------------------------------
// The given label's logit, fetched by one thread in two steps so that neither load is waited for at the row's end.
struct Label {
    uint32_t id;
    float x;
    __device__ __forceinline__ void load_id(const ScoreArgs &a, size_t row) { id = a.logprobs && threadIdx.x == 0 ? (uint32_t)a.labels[row] : 0xffffffffu; }
    template <class E>
    __device__ __forceinline__ void load_logit(const ScoreArgs &a, const typename E::raw *row) { x = id < a.C ? E::get(row[id]) : 0.0f; }
};
template <class E>
__device__ __forceinline__ void score_out(const ScoreArgs &a, size_t row, const Label &lab, const RowStats &st)
{
    if (threadIdx.x != 0) return;
    if (a.logprobs) a.logprobs[row] = lab.id < a.C ? logprob_of<E>(a, st, lab.x) : 0.0f;
    if (a.entropy) a.entropy[row] = st.ent;
    if (a.stats) a.stats[row] = make_float4(st.m, st.l2, st.ent, 0.0f);
}

// A piece of work: a row, or one of its segments.
struct Piece {
    size_t row;
    uint32_t first, n;
};
__device__ __forceinline__ Piece piece_of(size_t w, uint32_t segs, uint32_t seg, uint32_t C)
{
    const size_t row = segs == 1 ? w : w / segs;
    const uint32_t first = segs == 1 ? 0 : (uint32_t)(w - row * segs) * seg;
    return {row, first, C - first < seg ? C - first : seg};
}

// Without top classes: the row streams by, 64 or 128 bytes a thread in flight and 64 registers, so that eight blocks of 256 share a CU and
// every row of a 2048-row call is under way at once.  2048 x 131072 bfloat16: 83 us, 6.5 TB/s, where a kernel that only reads reaches 7.0; 7.4
// vector instructions a value (widen, maximum, multiply-add, exponential, two sums), at four cycles each 50 us, more for the exponential.
template <class E, int NT, bool PASSING>
__global__ __launch_bounds__(NT, 8) void score_kernel(ScoreArgs a)
{
    __shared__ LogitsLds sh;
    const size_t work = a.rows * a.segs;
    for (size_t w = blockIdx.x; w < work; w += gridDim.x) {
        const Piece p = piece_of(w, a.segs, a.seg, a.C);
        const typename E::raw *x = (const typename E::raw *)a.logits + p.row * a.stride;
        Label lab;
        if (a.segs == 1) lab.load_id(a, p.row);
        const Running r = scan_classes<E, NT, true, false, PASSING>(x + p.first, Span<E>(x + p.first, p.n), a.c, nullptr);
        if (a.segs == 1) lab.load_logit<E>(a, x);
        const float3 j = block_join<NT>(r, a.c, sh);
        if (a.segs > 1) {
            if (threadIdx.x == 0) a.part[w] = make_float4(j.x, j.y, j.z, 0.0f);
            continue;
        }
        score_out<E>(a, p.row, lab, row_ok(j) ? stats_of(j) : careful_stats<E, NT>(x, a.C, a.c, 0, sh));
    }
}

// With top classes: the row stays in registers, and blocks stay for many rows: once a row's candidates are found, the next row
// comes into the registers while they are ranked.  4096 x 32768 bfloat16, 64 classes: 78 us a pass, 3.4 TB/s, bound by the vector unit: 15.6
// instructions a value by the counters, 53 us at four cycles.  The scores' 7.4, two to look for candidates and about 150 a row and thread for
// threshold and ranking are 10.6 of them; where the others go is not known.
template <class E, int NT>
__global__ __launch_bounds__(NT, 4) void score_top_kernel(ScoreArgs a)
{
    __shared__ LogitsLds sh;
    __shared__ TopLds top;
    const size_t work = a.rows * a.segs;
    auto logits = [&](const Piece &p) { return (const typename E::raw *)a.logits + p.row * a.stride + p.first; };
    Resident<E, NT> reg;
    Piece p = piece_of(blockIdx.x, a.segs, a.seg, a.C);
    Span<E> span(logits(p), p.n);
    reg.template load<false>(logits(p), span);
    for (size_t w = blockIdx.x; w < work; w += gridDim.x) {
        const typename E::raw *x = logits(p);
        Label lab;
        if (a.segs == 1) lab.load_id(a, p.row);
        Running r = running_start(a.c);
        reg.each(span, [&](int, const float *v) { absorb<Resident<E, NT>::N, true>(v, a.c, r); });
        absorb<1, true>(&reg.edge, a.c, r);
        if (a.segs == 1) lab.load_logit<E>(a, x);
        reg.forget();
        const float3 j = block_join<NT>(r, a.c, sh);
        const bool ok = row_ok(j);
        RowStats st = {};
        uint32_t k = a.k;
        if (a.segs > 1) {
            if (threadIdx.x == 0) a.part[w] = make_float4(j.x, j.y, j.z, 0.0f);
            k = k < p.n ? k : p.n;                           // a short last segment fills up with keys below every class's
            for (uint32_t t = k + threadIdx.x; t < a.k; t += NT) a.part_key[w * a.k + t] = 0;
        } else {
            st = ok ? stats_of(j) : careful_stats<E, NT>(x, a.C, a.c, 0, sh);
            score_out<E>(a, p.row, lab, st);
        }
        const size_t row = p.row;
        const Span<E> now = span;
        const uint32_t first = p.first;
        auto next_row = [&] {
            if (w + gridDim.x >= work) return;
            p = piece_of(w + gridDim.x, a.segs, a.seg, a.C);
            span = Span<E>(logits(p), p.n);
            reg.template load<false>(logits(p), span);
        };
        top_classes<E, NT>(reg, x, now, first, k, r.m, ok, sh, top, next_row, [&](uint32_t rank, uint64_t key) {
            if (a.segs > 1) {
                a.part_key[w * a.k + rank] = key;
            } else {
                a.top_labels[row * a.k + rank] = (int32_t)top_index(key);
                a.top_logprobs[row * a.k + rank] = logprob_of<E>(a, st, top_value(key));
            }
        });
    }
}

// The shares of a split row put together, one block a row.  Latency only: 4.6 us for one row of 32 segments.
constexpr int JOIN_THREADS = 256;
template <class E>
__global__ __launch_bounds__(JOIN_THREADS) void score_join_kernel(ScoreArgs a)
{
    constexpr int NT = JOIN_THREADS;
    __shared__ LogitsLds sh;
    __shared__ TopLds top;
    for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const typename E::raw *x = (const typename E::raw *)a.logits + row * a.stride;
        // every load that depends on nothing else first
        Label lab;
        lab.load_id(a, row);
        const uint32_t n = a.segs * a.k;
        const uint64_t *keys = a.part_key + row * n;
        const uint64_t mine = threadIdx.x < n ? keys[threadIdx.x] : 0;
        float3 share = make_float3(M_START, 0.0f, 0.0f);     // (shares are about their exact maxima)
        for (uint32_t i = threadIdx.x; i < a.segs; i += NT) {
            const float4 p = a.part[row * a.segs + i];
            const float3 two[2] = {share, make_float3(p.x, p.y, p.z)};
            share = join(two, 2, a.c);
        }
        lab.load_logit<E>(a, x);
        const float M = wave_max(share.x);
        const float D = (share.x - M) * a.c, f = exp2_hw(D);
        const bool some = share.y != 0.0f;
        const float3 p = make_float3(M, wave_sum(some ? share.y * f : 0.0f), wave_sum(some ? __builtin_fmaf(D, share.y, share.z) * f : 0.0f));
        __syncthreads();
        if ((threadIdx.x & 63u) == 0) sh.part[threadIdx.x >> 6] = p;
        __syncthreads();
        const float3 j = join(sh.part, NT / WAVE, a.c);
        const RowStats st = row_ok(j) ? stats_of(j) : careful_stats<E, NT>(x, a.C, a.c, 0, sh);
        score_out<E>(a, row, lab, st);
        if (a.k) {
            uint32_t o = (uint32_t)(mine >> 24);
            for (uint32_t i = threadIdx.x + NT; i < n; i += NT) {
                const uint32_t q = (uint32_t)(keys[i] >> 24);
                o = q > o ? q : o;
            }
            const uint32_t G = top_groups(a.k), lanes = NT / G;
            for (uint32_t off = 1; off < lanes; off <<= 1) {
                const uint32_t q = __shfl_xor(o, off);
                o = q > o ? q : o;
            }
            __syncthreads();
            if (threadIdx.x % lanes == 0) top.group[threadIdx.x / lanes] = o;
            const uint32_t tau = top_threshold<NT>(G, a.k, sh, top);
            if (threadIdx.x < n && (uint32_t)(mine >> 24) >= tau) push_candidate(mine, sh, top);
            for (uint32_t i = threadIdx.x + NT; i < n; i += NT)
                if ((uint32_t)(keys[i] >> 24) >= tau) push_candidate(keys[i], sh, top);
            __syncthreads();
            const uint32_t got = sh.count;
            auto out = [&](uint32_t rank, uint64_t key) {
                a.top_labels[row * a.k + rank] = (int32_t)top_index(key);
                a.top_logprobs[row * a.k + rank] = logprob_of<E>(a, st, top_value(key));
            };
            if (got >= a.k && got <= TOP_CAP) {
                rank_candidates<NT>(got, a.k, top, out);
            } else {
                top_radix<NT>(n, a.k, sh, top, StoredKey{keys});
                for (uint32_t t = threadIdx.x; t < a.k; t += NT) out(t, top.key[t]);
            }
            __syncthreads();
        }
    }
}

// ------------------------------------------------------------------------------------------
// gradients
// ------------------------------------------------------------------------------------------
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

template <class E, int NT>
__device__ void zero_classes(typename E::raw *out, uint32_t n)
{
    constexpr int VEC = E::VEC;
    const uint32_t nvec = n / VEC;
    for (uint32_t i = threadIdx.x; i < nvec; i += NT) store_raw<E>(out + (size_t)i * VEC, u32x4{0, 0, 0, 0});
    if (threadIdx.x < n - nvec * VEC) out[nvec * VEC + threadIdx.x] = E::put(0.0f);
}

// out = p (ga + gb log2 p) at n classes of a row, p by the row's statistics.  Reads and writes go around the caches (nobody asks for either
// soon): 2048 x 131072 bfloat16 345 -> 312 us for the step.  Bound by memory: 186 us for 1.04 GB, 5.6 TB/s.
template <class E, int NT, int U, bool ENT>
__device__ __forceinline__ void write_grad(const RowStats &st, float ga, float gb, const typename E::raw *x, typename E::raw *out, uint32_t n, float c)
{
    constexpr int VEC = E::VEC;
    if (st.m == -INFINITY) {                                 // no class has any probability
        zero_classes<E, NT>(out, n);
        return;
    }
    auto value = [&](float v) {
        const float t = (v - st.m) * c - st.l2;
        return exp2_hw(t) * (ENT ? __builtin_fmaf(gb, vmax(t, T_FLOOR), ga) : ga);
    };
    const Span<E> span(x, n);
    const typename E::raw *body = x + span.head;
    typename E::raw *to = out + span.head;
    uint32_t i = threadIdx.x;
    for (; i + (U - 1) * NT < span.nvec; i += U * NT) {
        u32x4 w[U];
#pragma unroll
        for (int k = 0; k < U; ++k) w[k] = load_raw<E, true>(body + (size_t)(i + k * NT) * VEC);
#pragma unroll
        for (int k = 0; k < U; ++k) {
            float v[VEC];
            E::unpack(w[k], v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = value(v[e]);
            store_raw<E, true>(to + (size_t)(i + k * NT) * VEC, E::pack(v));
        }
    }
    for (; i < span.nvec; i += NT) {
        float v[VEC];
        E::unpack(load_raw<E, true>(body + (size_t)i * VEC), v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = value(v[e]);
        store_raw<E, true>(to + (size_t)i * VEC, E::pack(v));
    }
    if (threadIdx.x < span.edges) out[span.edge(threadIdx.x)] = E::put(value(E::get(x[span.edge(threadIdx.x)])));
}

template <class E, int NT, bool ENT>
__global__ __launch_bounds__(NT) void score_grad_kernel(ScoreGradArgs a)
{
    __shared__ LogitsLds sh;
    const size_t work = a.rows * a.segs;
    for (size_t w = blockIdx.x; w < work; w += gridDim.x) {
        const Piece p = piece_of(w, a.segs, a.seg, a.C);
        const typename E::raw *x = (const typename E::raw *)a.logits + p.row * a.stride;
        typename E::raw *out = (typename E::raw *)a.grad + p.row * a.C + p.first;
        const float4 f = a.stats[p.row];
        const RowStats st = {f.x, f.y, f.z, 0.0f};
        if (st.m == -INFINITY) {                             // an empty row has constant outputs
            zero_classes<E, NT>(out, p.n);
            continue;
        }
        const uint32_t n = a.k + 1;
        const float gh = ENT ? a.up_entropy[p.row] : 0.0f;
        __syncthreads();
        for (uint32_t j = threadIdx.x; j < n; j += NT) {
            int32_t id = -1;
            float v = 0.0f;
            if (j == a.k) {
                if (a.up_logprobs) id = a.labels[p.row], v = a.up_logprobs[p.row];
            } else
                id = a.top_labels[p.row * a.k + j], v = a.up_top[p.row * a.k + j];
            sh.id[j] = (uint32_t)id < a.C ? id : -1;
            sh.val[j] = (uint32_t)id < a.C ? v : 0.0f;
        }
        __syncthreads();
        float total = 0.0f;
        for (uint32_t j = 0; j < n; ++j) total += sh.val[j];
        // d/dx_i = (1/T) [ sum_j g_j [i = id_j] - p_i (G + gH (log p_i + H)) ]
        const float ga = -a.inv_t * (total + gh * st.ent), gb = -a.inv_t * gh * LN2;
        write_grad<E, NT, 16 / E::VEC, ENT>(st, ga, gb, x + p.first, out, p.n, a.c);
        __syncthreads();                                     // the block's own stores before the listed classes' (same addresses)
        for (uint32_t j = threadIdx.x; j < n; j += NT) {
            const uint32_t at = (uint32_t)sh.id[j] - p.first;
            float sum;
            if (sh.id[j] < 0 || at >= p.n || !first_entry(sh, j, n, sum)) continue;
            const float t = (E::get(x[sh.id[j]]) - st.m) * a.c - st.l2;
            out[at] = E::put(a.inv_t * sum + exp2_hw(t) * __builtin_fmaf(gb, vmax(t, T_FLOOR), ga));
        }
    }
}

// ------------------------------------------------------------------------------------------
// distillation
// ------------------------------------------------------------------------------------------
// The list of one row.  Renormalised: q = softmax of the teacher's values over the listed classes, and the statistics describe all of
// the student's classes.  Bucket: q = exp(teacher), the teacher's remaining mass q0 = 1 - sum q against the student's mass p0
// off the list, and the statistics describe the classes OFF the list; all classes follow by adding the listed ones, so neither
// p0 nor the rest's gradient suffers the cancellation of 1 - sum p.
//
// Everything that needs no statistics is done by the block's first wave while the row is on its way: entries lane and lane + 64.
struct ListEntries {
    int32_t id[2];       // -1: an unused place
    float t[2], x[2];

    // the two loads, the second with what the first has brought
    __device__ __forceinline__ void load_list(const DistillArgs &a, size_t row)
    {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t j = threadIdx.x + 64 * h;
            id[h] = -1;
            t[h] = -INFINITY;
            if (j < a.K) id[h] = a.ids[row * a.K + j], t[h] = a.teacher[row * a.K + j];
        }
    }
    template <class E>
    __device__ __forceinline__ void load_logits(const DistillArgs &a, const typename E::raw *row)
    {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            x[h] = -INFINITY;
            if ((uint32_t)id[h] < a.C) x[h] = E::get(row[id[h]]);
            else id[h] = -1, t[h] = -INFINITY;
        }
    }
};

// Fills sh.id (first entries of their classes; -1 otherwise), sh.val (a class's q, summed over its entries), sh.x (the student's
// logits there), sh.q and sh.logq (by entry) and sh.sum: sum q, q0, and for the bucket the listed classes' maximum and sum about it.
__device__ __forceinline__ void prepare_list(const DistillArgs &a, bool bucket, const ListEntries &en, LogitsLds &sh)
{
    const uint32_t lane = threadIdx.x;
    const bool on[2] = {en.id[0] >= 0, en.id[1] >= 0};
    float q[2] = {0.0f, 0.0f}, logq[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int h = 0; h < 2; ++h) sh.id[lane + 64 * h] = en.id[h];
    if (lane < 3) sh.id[128 + lane] = -1;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // (one wave's LDS accesses stay in order)
    float mass, q0 = 0.0f;
    if (!bucket) {
        const float tm = wave_max(vmax(en.t[0], en.t[1])), about = tm > -INFINITY ? tm : 0.0f;
        float e[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) e[h] = on[h] ? exp2_hw((en.t[h] - about) * LOG2E) : 0.0f;
        const float tt = wave_sum(e[0] + e[1]), logt = LN2 * log2_hw(tt);
        mass = tt == 0.0f ? 0.0f : tt == tt ? 1.0f : NAN;    // the maximum does not see a NaN, the sum does
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (tt != 0.0f) q[h] = e[h] / tt, logq[h] = (en.t[h] - about) - logt;
    } else {
        double sum = 0.0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            q[h] = on[h] ? exp_split(en.t[h]) : 0.0f;
            logq[h] = en.t[h];
            if (on[h]) sum += exp_wide(en.t[h]);
        }
        for (int off = 1; off < 64; off <<= 1) sum += __shfl_xor(sum, off);
        const double left = 1.0 - sum;           // exponentials and sum in double: where the list holds nearly everything, little is left of it
        q0 = left > 0.0 ? (float)left : left != left ? NAN : 0.0f;
        mass = (float)sum;
    }
    // entries of a class listed before
    bool first[2] = {on[0], on[1]}, twice = false;
    for (uint32_t i = 0; i < a.K; i += 4) {
        const int4 o = *(const int4 *)&sh.id[i];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t j = lane + 64 * h;
            const int32_t id = en.id[h];
            if ((o.x == id && i < j) || (o.y == id && i + 1 < j) || (o.z == id && i + 2 < j) || (o.w == id && i + 3 < j)) {
                twice |= first[h];
                first[h] = false;
            }
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t j = lane + 64 * h;
        sh.val[j] = sh.q[j] = q[h];
        sh.logq[j] = logq[h];
        sh.x[j] = en.x[h];
    }
    if (__any(twice)) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (!first[h]) continue;
            float sum = 0.0f;
            for (uint32_t i = 0; i < a.K; ++i)
                if (sh.id[i] == en.id[h]) sum += sh.q[i];
            sh.val[lane + 64 * h] = sum;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (!first[h]) sh.id[lane + 64 * h] = -1;
    }
    float top = -INFINITY, s = 0.0f;
    if (bucket) {
        top = wave_max(vmax(first[0] ? en.x[0] : -INFINITY, first[1] ? en.x[1] : -INFINITY));
        const float about = top > -INFINITY ? top : 0.0f;    // (a maximum of NaNs alone is -inf as well, their sum is NaN)
        s = wave_sum((first[0] ? exp2_hw((en.x[0] - about) * a.c) : 0.0f) + (first[1] ? exp2_hw((en.x[1] - about) * a.c) : 0.0f));
    }
    if (lane == 0) sh.sum[0] = mass, sh.sum[1] = q0, sh.sum[2] = top, sh.sum[3] = s;
}
template <class E>
__device__ __forceinline__ void load_and_prepare(const DistillArgs &a, bool bucket, size_t row, const typename E::raw *x, LogitsLds &sh)
{
    ListEntries en;
    en.load_list(a, row);
    en.load_logits<E>(a, x);
    prepare_list(a, bucket, en, sh);
}

// What follows once the streamed classes' statistics are there; the same in every thread.
struct ListTerms {
    float m, l2;         // all classes; m = -inf: none has any probability; NaN: so is the row
    float mass;          // sum q (+ q0)
    float dense;         // the gradient off the list, over coefficient and softmax of the streamed classes
    float rest;          // the bucket's part of the loss; NaN for a row that is
};
__device__ __forceinline__ ListTerms list_terms(const DistillArgs &a, bool bucket, const RowStats &st, const LogitsLds &sh)
{
    const float mass = sh.sum[0], q0 = sh.sum[1], top = sh.sum[2], s_on = sh.sum[3];
    ListTerms r = {st.m, st.l2, mass, mass, 0.0f};
    if (bucket) {
        const bool rest = st.m > -INFINITY;      // the bucket takes part
        if (rest) r.mass = mass + q0;
        r.m = vmax(st.m, top);
        r.l2 = -INFINITY;
        if (r.m > -INFINITY) {
            const float off = rest ? st.s * exp2_hw((st.m - r.m) * a.c) : 0.0f;
            const float on = top > -INFINITY ? s_on * exp2_hw((top - r.m) * a.c) : 0.0f;
            r.l2 = log2_hw(on + off);
            const BucketTerms b = bucket_terms(on, off, mass, q0, (st.m - r.m) * a.inv_t + LN2 * (st.l2 - r.l2));
            r.dense = b.dense;
            if (rest) r.rest = b.rest;
        }
    }
    // a NaN or +inf among the logits, also where nothing is listed, or among the teacher's values, except for an empty row
    if (st.m != st.m || s_on != s_on || (mass != mass && r.m > -INFINITY)) r.m = r.dense = r.rest = NAN;
    return r;
}

// Marks the listed classes among a span's, which starts at class `first`.
template <class E, int NT>
__device__ __forceinline__ void mask_listed(const DistillArgs &a, size_t row, uint32_t first, const Span<E> &span, uint32_t *mask)
{
    using M = Mask<E, NT>;
    const uint32_t words = M::words(span.nvec);
    __syncthreads();
    for (uint32_t i = threadIdx.x * 4; i < words; i += NT * 4) *(uint4 *)&mask[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    for (uint32_t j = threadIdx.x; j < a.K; j += NT) {
        const uint32_t at = (uint32_t)a.ids[row * a.K + j] - first;
        if (at >= span.n) continue;
        const uint32_t i = (at - span.head) / E::VEC;        // (classes of the head: far beyond nvec)
        if (at >= span.head && i < span.nvec) atomicOr(&mask[M::word(i)], 1u << (M::bit(i) + (at - span.head) % E::VEC));
        else atomicOr(&mask[words - 1], 1u << (at < span.head ? at : at - span.nvec * E::VEC));
    }
    __syncthreads();
}

// Loss of a row by the block's first wave.
__device__ __forceinline__ void loss_out(const DistillArgs &a, size_t row, float w, const RowStats &st, const ListTerms &r, const LogitsLds &sh)
{
    float terms = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t j = threadIdx.x + 64 * h;
        const float q = sh.q[j];
        if (q > 0.0f || q != q) terms += q * (sh.logq[j] - ((sh.x[j] - r.m) * a.inv_t - LN2 * r.l2));
    }
    terms = wave_sum(terms) + r.rest;
    if (threadIdx.x == 0) {
        a.out_rows[row] = r.m == -INFINITY ? 0.0f : w * a.t * a.t * terms;
        if (a.stats) a.stats[row] = make_float4(st.m, st.l2, st.s, 0.0f);
    }
}
__device__ __forceinline__ void ignored_out(const DistillArgs &a, size_t row)
{
    if (threadIdx.x != 0) return;
    a.out_rows[row] = 0.0f;
    if (a.stats) a.stats[row] = make_float4(-INFINITY, -INFINITY, 0.0f, 0.0f);
}
// The final values at the listed classes among the n from `first` on, over what the block has stored there.
template <class E, int NT>
__device__ __forceinline__ void listed_grad(const DistillArgs &a, float coef, const ListTerms &r, typename E::raw *out, uint32_t n, uint32_t first,
                                            const LogitsLds &sh)
{
    __syncthreads();                                         // the block's own stores first (same addresses)
    for (uint32_t j = threadIdx.x; j < a.K; j += NT) {
        const uint32_t at = (uint32_t)sh.id[j] - first;
        if (sh.id[j] >= 0 && at < n) out[at] = E::put(coef * (exp2_hw((sh.x[j] - r.m) * a.c - r.l2) * r.mass - sh.val[j]));
    }
    __syncthreads();
}

constexpr uint32_t MASK_CLASSES = 262144;        // of a bucket segment: 32 KB of mask

// Losses, one block per row or per segment of a row: the row streams by.  2048 x 32768 float32: 41.5 us, 6.1 TB/s.  The bucket's mask costs a
// word of LDS for every 32 values of a thread and, where a wave has a listed class in them, three more instructions a value: 2048 x
// 131072 bfloat16 ahead of a gradient, 64 listed 115 us, 4.4 TB/s, the same without the mask; why it stays below the scores' rate is not
// known.  (Eight blocks a CU for it: 312 -> 326 us with the gradient.)
template <class E, int NT, bool BUCKET, bool PASSING>
__global__ __launch_bounds__(NT, BUCKET ? 6 : 8) void distill_kernel(DistillArgs a)
{
    __shared__ LogitsLds sh;
    extern __shared__ __attribute__((aligned(16))) uint32_t mask[];
    const size_t work = a.rows * a.segs;
    for (size_t w = blockIdx.x; w < work; w += gridDim.x) {
        const Piece p = piece_of(w, a.segs, a.seg, a.C);
        const typename E::raw *x = (const typename E::raw *)a.logits + p.row * a.stride;
        const float weight = a.weights ? a.weights[p.row] : 1.0f;
        if (weight == 0.0f) {                                // ignored: 0 whatever it holds
            if (a.segs == 1) ignored_out(a, p.row);
            continue;
        }
        const Span<E> span(x + p.first, p.n);
        if (BUCKET) mask_listed<E, NT>(a, p.row, p.first, span, mask);
        if (a.segs == 1 && threadIdx.x < WAVE) load_and_prepare<E>(a, BUCKET, p.row, x, sh);
        const Running r = scan_classes<E, NT, false, BUCKET, PASSING>(x + p.first, span, a.c, mask);
        const float3 j = block_join<NT>(r, a.c, sh);
        if (a.segs > 1) {
            if (threadIdx.x == 0) a.part[w] = make_float4(j.x, j.y, 0.0f, 0.0f);
            continue;
        }
        const RowStats st = row_ok(j) ? stats_of(j) : careful_stats<E, NT>(x, a.C, a.c, BUCKET ? a.K : 0, sh);
        const ListTerms t = list_terms(a, BUCKET, st, sh);
        if (threadIdx.x < WAVE) loss_out(a, p.row, weight, st, t, sh);
        __syncthreads();
    }
}

// The shares of a split row put together, one wave a row.
template <class E>
__global__ __launch_bounds__(WAVE) void distill_join_kernel(DistillArgs a)
{
    __shared__ LogitsLds sh;
    for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const typename E::raw *x = (const typename E::raw *)a.logits + row * a.stride;
        const float weight = a.weights ? a.weights[row] : 1.0f;
        if (weight == 0.0f) {
            ignored_out(a, row);
            continue;
        }
        float3 share = make_float3(M_START, 0.0f, 0.0f);
        for (uint32_t i = threadIdx.x; i < a.segs; i += WAVE) {
            const float4 p = a.part[row * a.segs + i];
            const float3 two[2] = {share, make_float3(p.x, p.y, 0.0f)};
            share = join(two, 2, a.c);
        }
        load_and_prepare<E>(a, a.bucket, row, x, sh);
        const float M = wave_max(share.x);
        const float s = wave_sum(share.y != 0.0f ? share.y * exp2_hw((share.x - M) * a.c) : 0.0f);
        __syncthreads();
        const float3 j = make_float3(M, s, 0.0f);
        const RowStats st = row_ok(j) ? stats_of(j) : careful_stats<E, WAVE>(x, a.C, a.c, a.bucket ? a.K : 0, sh);
        loss_out(a, row, weight, st, list_terms(a, a.bucket, st, sh), sh);
        __syncthreads();
    }
}

// Losses and gradient of whole rows that fit into a block's registers: one read, one write.  (Fetching the next row's vectors as this
// row's gradients leave them was measured too: 4096 x 131072 bfloat16 433 -> 476 us.  Memory moves reads and writes faster apart.)
// Reads go around the caches, and writes where rows are long: 444 -> 431 us, 1024 rows 142 -> 128, 4096 x 30000 120 -> 104.
// 4096 x 131072 bfloat16: 427 us for 2.08 GB, 4.9 TB/s, what a copy of this size reaches.  One block of 1024 threads fills a CU's registers, so
// rows go in rounds of 256: a pass over 768 x 50021 float32 takes 80 us, 769 rows 88, 777 rows 90 to 92, 1024 rows 103.
// The list's terms take the form from the arguments: with BUCKET in its place the registers come out worse (renormalised 50 000 x 4000 bfloat16
// 187 -> 198 us, bucket 6000 x 30000 172 -> 178), where distill_kernel gains by it (2048 x 32768 float32 45.8 -> 41.4).
template <class E, int NT, bool BUCKET>
__global__ __launch_bounds__(NT, 4) void distill_fused_kernel(DistillArgs a)
{
    using Row = Resident<E, NT>;
    using M = Mask<E, NT>;
    constexpr int VEC = E::VEC;
    __shared__ LogitsLds sh;
    extern __shared__ __attribute__((aligned(16))) uint32_t mask[];
    for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const typename E::raw *x = (const typename E::raw *)a.logits + row * a.stride;
        typename E::raw *out = (typename E::raw *)a.grad + row * a.C;
        const float weight = a.weights ? a.weights[row] : 1.0f;
        if (weight == 0.0f) {                                // ignored: 0 whatever it holds
            ignored_out(a, row);
            zero_classes<E, NT>(out, a.C);
            continue;
        }
        ListEntries en;
        if (threadIdx.x < WAVE) en.load_list(a, row);
        const Span<E> span(x, a.C);
        Row reg;
        reg.template load<true>(x, span);
        if (BUCKET) mask_listed<E, NT>(a, row, 0, span, mask);
        if (threadIdx.x < WAVE) en.load_logits<E>(a, x);
        Running run = running_start(a.c);
        reg.each(span, [&](int k, const float *v) {
            if (BUCKET) {
                const uint32_t b = mask[M::word(k * NT + reg.tid)] >> M::bit(k * NT);
                float u[Row::N];
#pragma unroll
                for (int j = 0; j < Row::N; ++j) u[j] = v[j];
                if (__any(b & ((1u << Row::N) - 1)))
#pragma unroll
                    for (int j = 0; j < Row::N; ++j) u[j] = b >> j & 1u ? -INFINITY : u[j];
                absorb<Row::N, false>(u, a.c, run);
            } else
                absorb<Row::N, false>(v, a.c, run);
        });
        float edge = reg.edge;
        if (BUCKET && reg.tid < span.edges && mask[M::words(span.nvec) - 1] >> reg.tid & 1u) edge = -INFINITY;
        absorb<1, false>(&edge, a.c, run);
        reg.forget();
        if (threadIdx.x < WAVE) prepare_list(a, a.bucket, en, sh);
        const float3 j = block_join<NT>(run, a.c, sh);
        const RowStats st = row_ok(j) ? stats_of(j) : careful_stats<E, NT>(x, a.C, a.c, BUCKET ? a.K : 0, sh);
        const ListTerms t = list_terms(a, a.bucket, st, sh);
        if (threadIdx.x < WAVE) loss_out(a, row, weight, st, t, sh);
        const float coef = weight * a.t * a.scale, dense = coef * t.dense;
        const bool none = t.m == -INFINITY || (st.m == -INFINITY && t.m == t.m);     // nothing has a probability, or nothing off the list
        auto value = [&](float v) { return none ? 0.0f : exp2_hw((v - st.m) * a.c - st.l2) * dense; };
        typename E::raw *to = out + span.head;
#pragma unroll
        for (int k = 0; k < Row::R; ++k) {
            const uint32_t i = k * NT + reg.tid;
            if (i < span.nvec) {
                float v[VEC];
                E::unpack(reg.w[k], v);
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[e] = value(v[e]);
                store_raw<E, NT == 1024>(to + (size_t)i * VEC, E::pack(v));
            }
        }
        if (reg.tid < span.edges) out[span.edge(reg.tid)] = E::put(value(reg.edge));
        if (t.m != -INFINITY) listed_grad<E, NT>(a, coef, t, out, a.C, 0, sh);
        else __syncthreads();
    }
}

// The gradient from the statistics of an earlier launch, one block per row or per segment of a row (write_grad has the figures).
template <class E, int NT>
__global__ __launch_bounds__(NT) void distill_grad_kernel(DistillArgs a)
{
    __shared__ LogitsLds sh;
    const size_t work = a.rows * a.segs;
    for (size_t w = blockIdx.x; w < work; w += gridDim.x) {
        const Piece p = piece_of(w, a.segs, a.seg, a.C);
        const typename E::raw *x = (const typename E::raw *)a.logits + p.row * a.stride;
        typename E::raw *out = (typename E::raw *)a.grad + p.row * a.C + p.first;
        const float weight = a.weights ? a.weights[p.row] : 1.0f;
        if (weight == 0.0f) {
            zero_classes<E, NT>(out, p.n);
            continue;
        }
        if (threadIdx.x < WAVE) load_and_prepare<E>(a, a.bucket, p.row, x, sh);
        __syncthreads();
        const float4 f = a.stats[p.row];
        RowStats st = {f.x, f.y, 0.0f, f.z};
        const ListTerms t = list_terms(a, a.bucket, st, sh);
        if (t.m != t.m) st.m = t.m;                          // NaN off the list too, where nothing there has a probability
        const float coef = weight * a.t * a.scale * (a.up ? a.up[a.up_rows ? p.row : 0] : 1.0f);
        if (t.m == -INFINITY) {
            zero_classes<E, NT>(out, p.n);
            __syncthreads();
            continue;
        }
        write_grad<E, NT, 16 / E::VEC, false>(st, coef * t.dense, 0.0f, x + p.first, out, p.n, a.c);
        listed_grad<E, NT>(a, coef, t, out, p.n, p.first, sh);
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
    if (rows > (size_t)1 << 32 || stride > (size_t)1 << 40) return fail(ODBOX_EINVAL, "%s: rows over 2^32 or row_stride over 2^40", name);
    if (!(temperature >= 1e-6f && temperature <= 1e6f)) return fail(ODBOX_EINVAL, "%s: temperature %g is not in 1e-6..1e6", name, (double)temperature);
    if (rows && !logits) return fail(ODBOX_EINVAL, "%s: NULL logits", name);
    if ((uintptr_t)logits % (dtype == ODBOX_DTYPE_F32 ? 4 : 2)) return fail(ODBOX_EINVAL, "%s: logits are not aligned to their element", name);
    return 0;
}

// How a row's classes are dealt out to blocks: whole rows where there are enough of them to fill the chip, else segments of at
// least 4096 classes so that about `blocks` blocks run.  A segment is a multiple of 8 classes and holds at most `most`.
struct Split {
    uint32_t segs, seg;
};
static Split split_rows(size_t rows, uint32_t C, uint32_t blocks, uint32_t most)
{
    if (rows == 0) return {1, C};
    uint32_t segs = rows >= blocks ? 1 : (uint32_t)((blocks + rows - 1) / rows);
    const uint32_t fit = C / 4096 ? C / 4096 : 1, need = (C + most - 1) / most;
    segs = segs < fit ? segs : fit;
    segs = segs > need ? segs : need;
    uint32_t seg = segs == 1 ? C : (((C + segs - 1) / segs + 7) & ~7u);
    if (seg > most && segs > 1) seg = most;
    return {(C + seg - 1) / seg, seg};
}
constexpr uint32_t FILL_BLOCKS = 1024;
// Loss and gradient by whole rows from this many on; few rows fill the chip better in segments.  Whole rows / segments, us a pass: bucket, 50021
// float32 classes, 300 rows 45.4 / 45.2, 520 rows 69.1 / 67.2, 768 rows 80.3 / 89.3, 777 rows 92.5 / 91.4; renormalised 520 rows 60.1 / 66.0, 777 rows
// 82.7 / 90.6; 520 rows of 9000 classes 17.0 / 24.5.  (Renormalised 200 rows take 23.0 / 32.8: the limit could be lower.)
constexpr size_t FUSE_ROWS = 512;
// What a block of NT threads holds in registers.
static uint32_t resident(int dtype, int nt) { return 16u * nt * (dtype == ODBOX_DTYPE_F32 ? 4 : 8); }
// With top classes a segment fits 256 threads' registers, however many rows there are: blocks of 1024 threads wait longer at their
// barriers than the join takes (2048 x 131072 bfloat16, 20 classes 155 / 191 us; 4096 x 50000, 8 classes 133 / 206 us).
static Split score_split(size_t rows, uint32_t C, int k, int dtype) { return split_rows(rows, C, FILL_BLOCKS, k ? resident(dtype, 256) : 1u << 24); }
static Split distill_split(size_t rows, uint32_t C)
{
    return split_rows(rows, C, FILL_BLOCKS, MASK_CLASSES);
}
// Logits that pass by once (no statistics are kept for a gradient) are read around the caches from the Infinity Cache's own size on, 256 MB.
// Below, it is a loss where they are still in the cache and a gain where they are not.  Cached / around, us, the same logits each time, and two sets of
// them in turn: scores of 50021 bfloat16 classes, 96 MB 24.5 / 23.4 and 23.4 / 24.0; 192 MB 33.3 / 34.4 and 39.3 / 35.7; 240 MB 42.2 / 43.9 and 49.1 / 44.4;
// 256 MB 44.7 / 46.0 and 51.4 / 46.6; 288 MB 50.0 / 50.0 and 56.2 / 51.2; 512 MB 94.8 / 85.7 and 94.0 / 86.2.  Losses of 32768 float32 classes, 192 MB 33.2 / 33.4
// and 38.6 / 34.1; 256 MB 42.0 / 42.8 and 49.2 / 43.4; 512 MB 93.7 / 82.4 and 93.6 / 82.9.  Ahead of a gradient the same
// loads cost what its second read then misses (1021 x 100003 float16 scores both ways 126 -> 146 us, 4600 rows still 590 -> 618); losses
// gain where the cache holds little of them: both ways 300 x 1000003 bfloat16 (600 MB) 376 -> 384 us, 3600 x 100003 (720 MB) 455 ->
// 442, 4000 x 131072 605 -> 554.
static bool passes(size_t rows, int C, int dtype, size_t from) { return rows * C >= from / (dtype == ODBOX_DTYPE_F32 ? 4 : 2); }
constexpr size_t PASS_ONCE = (size_t)256 << 20, PASS_AGAIN = (size_t)640 << 20;
// Whole rows that 64 threads could hold in registers get a wave each, which waits for nobody (256 threads / a wave: scores of 100 000 x
// 2100 bfloat16 189 / 98 us, of 30 000 x 8000 100 / 87; losses of 50 000 x 4000 float32 188 / 119; a bucket step of 50 000 x 4000 bfloat16
// 719 / 360).
#define BY_WIDTH(dtype, sp, ...)                                                            \
    do {                                                                                    \
        if ((sp).segs == 1 && (sp).seg <= resident(dtype, 64)) { constexpr int NT = 64; __VA_ARGS__; } \
        else { constexpr int NT = 256; __VA_ARGS__; }                                       \
    } while (0)
// Blocks that stay: as many as the 256 CUs hold at four waves a SIMD (128 registers).
static dim3 staying_grid(size_t work, int nt)
{
    const size_t fit = 256 * (1024 / nt);
    return dim3((uint32_t)(work < fit ? work : fit));
}
// f(integral_constant): the smallest block that holds n classes in registers
template <class F>
static void resident_variant(int dtype, uint32_t n, F f)
{
    if (n <= resident(dtype, 64)) f(std::integral_constant<int, 64>());
    else if (n <= resident(dtype, 256)) f(std::integral_constant<int, 256>());
    else f(std::integral_constant<int, 1024>());
}

}  // namespace odbox

using namespace odbox;

extern "C" {

size_t odbox_label_logprobs_workspace(size_t rows, int C, int top_k)
{
    if (C < 1 || top_k < 0) return 0;
    const Split sp = score_split(rows, (uint32_t)C, top_k, ODBOX_DTYPE_F32);       // (float32 has the most segments)
    return sp.segs == 1 ? 0 : rows * sp.segs * (sizeof(float4) + (size_t)top_k * sizeof(uint64_t));
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
    if (!aligned16(workspace)) return fail(ODBOX_EINVAL, "%s: workspace must be 16-byte aligned", name);
    const Split sp = score_split(rows, (uint32_t)C, top_k, dtype);
    if (sp.segs > 1 && !workspace) return fail(ODBOX_EINVAL, "%s: NULL workspace", name);
    float4 *part = (float4 *)workspace;
    ScoreArgs a = {logits, rows, row_stride, (uint32_t)C, (uint32_t)top_k, LOG2E / temperature, 1.0f / temperature, labels, out_logprobs,
                   out_entropy, out_top_logprobs, out_top_labels, (float4 *)out_stats, sp.segs, sp.seg, part,
                   (uint64_t *)(part + (sp.segs > 1 ? rows * sp.segs : 0))};
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid = work_grid(rows * sp.segs);
    if (score_is_short(dtype, C, top_k)) {
        score_short(dtype, a, st);
        return launch_status(name);
    }
    if (top_k && sp.seg <= resident(dtype, 64)) LOGITS_LAUNCH(dtype, (score_top_kernel<E, 64>), staying_grid(rows * sp.segs, 64), dim3(64), 0, st, a);
    else if (top_k) LOGITS_LAUNCH(dtype, (score_top_kernel<E, 256>), staying_grid(rows * sp.segs, 256), dim3(256), 0, st, a);
    else if (!out_stats && passes(rows, C, dtype, PASS_ONCE)) BY_WIDTH(dtype, sp, LOGITS_LAUNCH(dtype, (score_kernel<E, NT, true>), grid, dim3(NT), 0, st, a));
    else BY_WIDTH(dtype, sp, LOGITS_LAUNCH(dtype, (score_kernel<E, NT, false>), grid, dim3(NT), 0, st, a));
    if (sp.segs > 1) LOGITS_LAUNCH(dtype, score_join_kernel<E>, work_grid(rows), dim3(JOIN_THREADS), 0, st, a);
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
    const Split sp = score_split(rows, (uint32_t)C, 0, dtype);
    ScoreGradArgs a = {logits, rows, row_stride, (uint32_t)C, (uint32_t)(upstream_top ? top_k : 0), LOG2E / temperature, 1.0f / temperature,
                       labels, top_labels, (const float4 *)stats, upstream_logprobs, upstream_entropy, upstream_top, grad, sp.segs, sp.seg};
    const dim3 grid = work_grid(rows * sp.segs);
    if (C <= short_limit(dtype)) {
        score_grad_short(dtype, a, (hipStream_t)stream);
        return launch_status(name);
    }
    if (upstream_entropy) BY_WIDTH(dtype, sp, LOGITS_LAUNCH(dtype, (score_grad_kernel<E, NT, true>), grid, dim3(NT), 0, (hipStream_t)stream, a));
    else BY_WIDTH(dtype, sp, LOGITS_LAUNCH(dtype, (score_grad_kernel<E, NT, false>), grid, dim3(NT), 0, (hipStream_t)stream, a));
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
    (void)K;
    if (C < 1) return 0;
    // blocks of the sum, row losses, row statistics and shares of split rows
    const Split sp = distill_split(rows, (uint32_t)C);
    return SUM_BLOCKS * sizeof(double) + ((rows + 3) / 4) * 4 * sizeof(float) + rows * sizeof(float4) + (sp.segs > 1 ? rows * sp.segs * sizeof(float4) : 0);
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
    const bool is_short = C <= short_limit(dtype);
    const bool fused = grad && !is_short && rows >= FUSE_ROWS && (uint32_t)C <= resident(dtype, 1024);
    const Split sp = fused ? Split{1, (uint32_t)C} : distill_split(rows, (uint32_t)C);
    float4 *spare = (float4 *)((float *)(partial + SUM_BLOCKS) + (rows + 3) / 4 * 4);
    float4 *keep = out_stats ? (float4 *)out_stats : grad && !is_short && !fused ? spare : nullptr;
    DistillArgs a = {logits, rows, row_stride, (uint32_t)C, (uint32_t)K, LOG2E / temperature, temperature, 1.0f / temperature, scale, rest,
                     teacher_logprobs, teacher_labels, row_weights, per_row, keep, nullptr, 0, grad, sp.segs, sp.seg, spare + rows};
    const dim3 grid = work_grid(rows * sp.segs);
    // Mask::words for NT threads, and what clearing them by fours may add
    const auto mask_bytes = [&](uint32_t nt) { return rest == ODBOX_REST_BUCKET ? ((size_t)(sp.seg + 32 * nt - 1) / (32 * nt) * nt + 4) * 4 : 0; };
    if (is_short) {
        distill_short(dtype, rest, grad, a, st);
    } else if (fused) {
        resident_variant(dtype, (uint32_t)C, [&](auto nt) {
            constexpr int NT = decltype(nt)::value;
            if (rest == ODBOX_REST_BUCKET) LOGITS_LAUNCH(dtype, (distill_fused_kernel<E, NT, true>), staying_grid(rows, NT), dim3(NT), mask_bytes(NT), st, a);
            else LOGITS_LAUNCH(dtype, (distill_fused_kernel<E, NT, false>), staying_grid(rows, NT), dim3(NT), 0, st, a);
        });
    } else {
        const bool passing = passes(rows, C, dtype, keep ? PASS_AGAIN : PASS_ONCE);
        if (rest == ODBOX_REST_BUCKET) {
            if (passing) BY_WIDTH(dtype, sp, LOGITS_LAUNCH(dtype, (distill_kernel<E, NT, true, true>), grid, dim3(NT), mask_bytes(NT), st, a));
            else BY_WIDTH(dtype, sp, LOGITS_LAUNCH(dtype, (distill_kernel<E, NT, true, false>), grid, dim3(NT), mask_bytes(NT), st, a));
        } else {
            if (passing) BY_WIDTH(dtype, sp, LOGITS_LAUNCH(dtype, (distill_kernel<E, NT, false, true>), grid, dim3(NT), 0, st, a));
            else BY_WIDTH(dtype, sp, LOGITS_LAUNCH(dtype, (distill_kernel<E, NT, false, false>), grid, dim3(NT), 0, st, a));
        }
        if (sp.segs > 1) LOGITS_LAUNCH(dtype, distill_join_kernel<E>, work_grid(rows), dim3(WAVE), 0, st, a);
        if (grad) BY_WIDTH(dtype, sp, LOGITS_LAUNCH(dtype, (distill_grad_kernel<E, NT>), grid, dim3(NT), 0, st, a));
    }
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
    const Split sp = distill_split(rows, (uint32_t)C);
    DistillArgs a = {logits, rows, row_stride, (uint32_t)C, (uint32_t)K, LOG2E / temperature, temperature, 1.0f / temperature, scale, rest, teacher_logprobs,
                     teacher_labels, row_weights, nullptr, (float4 *)stats, upstream, upstream_rows, grad, sp.segs, sp.seg, nullptr};
    if (C <= short_limit(dtype)) {
        distill_short(dtype, rest, true, a, (hipStream_t)stream);
    } else
        BY_WIDTH(dtype, sp, LOGITS_LAUNCH(dtype, (distill_grad_kernel<E, NT>), work_grid(rows * sp.segs), dim3(NT), 0, (hipStream_t)stream, a));
    return launch_status("distill_loss_backward");
}

}  // extern "C"
