// token_loss.cu - kernels of the token log-probabilities and of the losses
// made of them (include/quasar_losses.h).
//
// The mathematics: with k = log2(e) / T, M the largest logit of a row, R = M*k
// rounded to a whole number and t = l*k - R (one fused multiply-add), the row's
// softmax needs S = sum 2^t and its entropy also Q = sum 2^t * t:
//   logprob = ln2 * t_target - ln S,  entropy = ln S - ln2 * Q / S,
//   p_v = 2^t / S.
// M is not known while the row streams, so a thread sums against a reference
// that trails its running maximum and moves (one rescale of the sums) only
// when a logit passes it by 2^LAG: terms stay below 2^LAG, far inside fp32,
// and rescales are rare. A row whose |M|*k passes 2^24 (masked throughout by a
// large negative value) is summed over again with t = (l - M) * k.
//
// What bounds it: HBM for fp32 (4 bytes an element and pass); for 16-bit
// types one exponential per element and pass on the special-function unit
// (16 a clock and SM) takes 0.7 of the time that the bytes take.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "ptx.cuh"
#include "token_loss.cuh"

namespace qs {
namespace loss {

constexpr int U = 4;           // 16-byte loads in flight per thread
constexpr int MAXC = 8;        // CTAs of a row's cluster at most (the portable limit)
constexpr float LAG = 20.0f;   // powers of two that a term may stand above the reference
// l * k - c is good to a fraction of 1 only while l * k is below 2^24 or so:
// rows whose |M| * k reaches that are summed with differences taken first, and
// no reference goes below it (masked logits of -1e9 or -1e30 end at 2^t = 0).
constexpr float WIDE = 16777216.0f;
constexpr float NEG = -WIDE;
constexpr double LN2 = 0.6931471805599453094;

template <typename T>
struct Type;
template <>
struct Type<float> {
    static constexpr int N = 4;  // elements of a 16-byte pack
    static constexpr uint32_t NEG_INF = 0xFF800000u;
};
template <>
struct Type<__half> {
    static constexpr int N = 8;
    static constexpr uint32_t NEG_INF = 0xFC00FC00u;
};
template <>
struct Type<__nv_bfloat16> {
    static constexpr int N = 8;
    static constexpr uint32_t NEG_INF = 0xFF80FF80u;
};

__device__ __forceinline__ float widen1(float x) { return x; }
__device__ __forceinline__ float widen1(__half x) { return __half2float(x); }
__device__ __forceinline__ float widen1(__nv_bfloat16 x) { return __bfloat162float(x); }

// A pack's elements in fp32, in order.
__device__ __forceinline__ void widen(const uint4& p, float (&x)[4], float*) {
    x[0] = __uint_as_float(p.x), x[1] = __uint_as_float(p.y), x[2] = __uint_as_float(p.z), x[3] = __uint_as_float(p.w);
}
__device__ __forceinline__ void widen(const uint4& p, float (&x)[8], __nv_bfloat16*) {
    const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int i = 0; i < 4; i++) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
}
__device__ __forceinline__ void widen(const uint4& p, float (&x)[8], __half*) {
    const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
}

__device__ __forceinline__ uint4 narrow(const float (&x)[4], float*) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
}
__device__ __forceinline__ uint4 narrow(const float (&x)[8], __nv_bfloat16*) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(x[2 * i + 1]), "f"(x[2 * i]));
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 narrow(const float (&x)[8], __half*) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(x[2 * i + 1]), "f"(x[2 * i]));
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void put1(float* p, float x) { *p = x; }
__device__ __forceinline__ void put1(__half* p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void put1(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// Plain loads (not .nc): the gradient may be written over the logits.
__device__ __forceinline__ uint4 load_pack(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// A row as whole 16-byte packs with ragged edges: the first `head` elements
// come before the first 16-byte boundary, then `packs` packs, then `tail`.
struct Span {
    int head, packs, tail;
};
template <typename T>
__device__ __forceinline__ Span span_of(const T* row, int V) {
    const int off = (int)(((uintptr_t)row & 15) / sizeof(T));
    Span s;
    s.head = min(V, off ? Type<T>::N - off : 0);
    s.packs = (V - s.head) / Type<T>::N;
    s.tail = V - s.head - s.packs * Type<T>::N;
    return s;
}


// Part `part` of `parts` of a row's packs, and the edge element (of part 0)
// that thread tid takes: at most 2 * (N - 1) of them, one a thread.
struct Slice {
    int head, lo, n;  // packs [lo, lo + n)
    int edge;         // element, or -1
};
template <typename T>
__device__ __forceinline__ Slice slice_of(const T* row, int V, int part, int parts, int tid) {
    const Span sp = span_of(row, V);
    Slice s;
    s.head = sp.head;
    s.lo = (int)((unsigned)sp.packs * (unsigned)part / (unsigned)parts);
    s.n = (int)((unsigned)sp.packs * (unsigned)(part + 1) / (unsigned)parts) - s.lo;
    s.edge = part == 0 && tid < sp.head + sp.tail ? (tid < sp.head ? tid : V - sp.tail + (tid - sp.head)) : -1;
    return s;
}

// Largest element of some packs (NaN is left to the sums).
template <int P>
__device__ __forceinline__ float packs_max(const uint4 (&p)[P], float*) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < P; i++) {
        m = max3(m, __uint_as_float(p[i].x), __uint_as_float(p[i].y));
        m = max3(m, __uint_as_float(p[i].z), __uint_as_float(p[i].w));
    }
    return m;
}
#define QS_MAX2(op, d, a, b) asm(op " %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b))
template <int P>
__device__ __forceinline__ float packs_max(const uint4 (&p)[P], __nv_bfloat16*) {
    uint32_t m = Type<__nv_bfloat16>::NEG_INF;
#pragma unroll
    for (int i = 0; i < P; i++) {
        uint32_t a, b;
        QS_MAX2("max.bf16x2", a, p[i].x, p[i].y);
        QS_MAX2("max.bf16x2", b, p[i].z, p[i].w);
        QS_MAX2("max.bf16x2", a, a, b);
        QS_MAX2("max.bf16x2", m, m, a);
    }
    return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xFFFF0000u));
}
template <int P>
__device__ __forceinline__ float packs_max(const uint4 (&p)[P], __half*) {
    uint32_t m = Type<__half>::NEG_INF;
#pragma unroll
    for (int i = 0; i < P; i++) {
        uint32_t a, b;
        QS_MAX2("max.f16x2", a, p[i].x, p[i].y);
        QS_MAX2("max.f16x2", b, p[i].z, p[i].w);
        QS_MAX2("max.f16x2", a, a, b);
        QS_MAX2("max.f16x2", m, m, a);
    }
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&m));
    return fmaxf(f.x, f.y);
}
#undef QS_MAX2

// ---- running sums of one thread -------------------------------------------

struct Acc {
    float c;     // scaled reference that the sums are taken against (NEG: none yet)
    float mx;    // largest element
    f32x2 s, q;  // sums of 2^t and of 2^t * t, t = l * k - c, in two lanes
};

__device__ __forceinline__ Acc acc_new() { return Acc{NEG, -INFINITY, pack2(0.0f, 0.0f), pack2(0.0f, 0.0f)}; }

// Moves the reference up to the scaled maximum of what comes next.
template <bool ENT>
__device__ __forceinline__ void acc_raise(Acc& a, float mx, float k) {
    a.mx = fmaxf(a.mx, mx);
    if (fmaf(mx, k, -a.c) > LAG) {
        const float c = rintf(mx * k), d = fmaxf(a.c - c, -1e30f);  // finite, for sums still at 0
        const float f = ex2_approx(d);
        const f32x2 ff = pack2(f, f);
        if (ENT) a.q = mul2(fma2(a.s, pack2(d, d), a.q), ff);
        a.s = mul2(a.s, ff);
        a.c = c;
    }
}

template <bool ENT, int N>
__device__ __forceinline__ void acc_add(Acc& a, const float (&x)[N], float k) {
    const f32x2 nc = pack2(-a.c, -a.c), kk = pack2(k, k);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const f32x2 t = fma2(pack2(x[i], x[i + 1]), kk, nc);
        float t0, t1;
        unpack2(t, t0, t1);
        const f32x2 e = pack2(ex2_approx(t0), ex2_approx(t1));
        a.s = add2(a.s, e);
        // a term of 0 at t = -inf must not become NaN; NaN stays in e
        if (ENT) a.q = fma2(e, pack2(fmaxf(t0, -200.0f), fmaxf(t1, -200.0f)), a.q);
    }
}

template <typename T, bool ENT, int P>
__device__ __forceinline__ void acc_packs(Acc& a, const uint4 (&p)[P], float k) {
    acc_raise<ENT>(a, packs_max(p, (T*)nullptr), k);
#pragma unroll
    for (int i = 0; i < P; i++) {
        float x[Type<T>::N];
        widen(p[i], x, (T*)nullptr);
        acc_add<ENT>(a, x, k);
    }
}

template <bool ENT>
__device__ __forceinline__ void acc_one(Acc& a, float x, float k) {
    const float y[2] = {x, -INFINITY};
    acc_raise<ENT>(a, x, k);
    acc_add<ENT>(a, y, k);
}

// (max, sum, Q) of a set of elements, the sums against the scaled maximum.
struct __align__(16) Part {
    float m, s, q, tag;
};

// The reference of sums with maximum m (finite for a maximum of the lowest
// value or -inf, whose sums are 0).
__device__ __forceinline__ float scaled(float m, float k) { return fmaxf(rintf(m * k), NEG); }

// Brings sums taken against the scaled reference `from` to the one of `m`.
__device__ __forceinline__ void rebase(float& s, float& q, float from, float m, float k) {
    const float d = fmaxf(from - scaled(m, k), -1e30f);
    const float f = ex2_approx(d);
    q = fmaf(s, d, q) * f;
    s *= f;
}

template <bool ENT>
__device__ __forceinline__ Part warp_part(const Acc& a, float k) {
    Part p;
    p.m = warp_max(a.mx);
    float s0, s1, q0, q1;
    unpack2(a.s, s0, s1);
    unpack2(a.q, q0, q1);
    s0 += s1, q0 += q1;
    rebase(s0, q0, a.c, p.m, k);
    p.s = warp_sum(s0);
    p.q = ENT ? warp_sum(q0) : 0.0f;
    p.tag = 0.0f;
    return p;
}

// A row's joined sums: 2^(l * k - R) over the row adds to S.
struct Row {
    float M;
    double S, Q, R;
    bool wide;
};

// One warp joins n parts, in the same order in every warp.
template <bool ENT>
__device__ __forceinline__ Row join_parts(const Part* parts, int n, float k) {
    const int lane = threadIdx.x & 31;
    Row w;
    w.M = -INFINITY;
    for (int i = lane; i < n; i += 32) w.M = fmaxf(w.M, parts[i].m);
    w.M = warp_max(w.M);
    float s = 0.0f, q = 0.0f;
    for (int i = lane; i < n; i += 32) {
        Part p = parts[i];
        rebase(p.s, p.q, scaled(p.m, k), w.M, k);
        s += p.s, q += p.q;
    }
    w.S = warp_sum((double)s);
    w.Q = ENT ? warp_sum((double)q) : 0.0;
    const float c = scaled(w.M, k);
    w.R = (double)c;
    w.wide = !(fabsf(c) < WIDE) && !isinf(w.M);
    return w;
}

// ---- one row's scalars ------------------------------------------------------

// grad_v = 2^(l * k - c) * (a + b * (l * k - c)) + [v == target] * one
struct Coef {
    float c, a, b, one;
    float lt;  // the target's logit
    int kind;  // ROW_*
};
// ROW_WIDE: c is M itself, t = (l - c) * k, and elements of p = 0 have a gradient
// of 0 whatever a and b (rows of infinite derivatives are taken so, too).
enum { ROW_SUM = 0, ROW_ZERO = 1, ROW_NAN = 2, ROW_WIDE = 3 };

constexpr float STEEP = 1e38f;  // a coefficient beyond this counts as infinite
__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// The gradient of g_lp * logprob + g_ent * entropy: p_v = 2^t / S and
// ln p_v = ln2 * t - ln S, so (g_lp ([v==target] - p) - g_ent p (ln p + H)) / T
// has the form of Coef, with H - ln S = -ln2 * Q / S. Where both derivatives
// are 0 (a clipped ratio) the row's gradient is zeros, without its logits.
__device__ __forceinline__ Coef make_coef(float M, float R, bool wide, float S, float h_ln_s, float g_lp, float g_ent, float inv_t) {
    Coef o;
    const float w = -inv_t / S;
    o.c = wide ? M : R;
    o.a = w * (g_lp + (g_ent != 0.0f ? g_ent * h_ln_s : 0.0f));
    o.b = w * (float)LN2 * g_ent;
    o.one = g_lp * inv_t;
    o.lt = 0.0f;
    o.kind = (g_lp == 0.0f && g_ent == 0.0f) || (M == -INFINITY && S == S) ? ROW_ZERO : wide ? ROW_WIDE : ROW_SUM;
    if (!(fabsf(o.a) <= STEEP && fabsf(o.b) <= STEEP) && o.kind != ROW_ZERO) {
        o.kind = o.a == o.a && o.b == o.b ? ROW_WIDE : ROW_NAN;  // NaN of S or of a derivative
        o.c = M;
        if (fabsf(o.a) > STEEP) o.a *= INFINITY;
        if (fabsf(o.b) > STEEP) o.b *= INFINITY;
    }
    return o;
}
// A row without an element-wise gradient.
__device__ __forceinline__ Coef fill_coef(bool nan) {
    Coef o;
    o.c = o.a = o.b = o.one = o.lt = 0.0f;
    o.kind = nan ? ROW_NAN : ROW_ZERO;
    return o;
}

// The target's logit as its gradient takes it: nothing beside an infinite derivative.
__device__ __forceinline__ float target_logit(const Coef& c, float l) { return finite(c.one) ? l : -INFINITY; }

struct RowIn {  // a row's inputs beside its logits
    float lt, adv, old_lp, ref_lp;
    double weight;
};

// ln S to about 3e-8 absolute: the exponent's part in 64 bits, the mantissa's
// by logf on [1, 2).
__device__ __forceinline__ double ln_sum(double S) {
    const float s = (float)S;
    if (!(s > 1e-30f && s < 1e30f)) return (double)logf(s);
    const int e = ((__float_as_int(s) >> 23) & 255) - 127;
    const float m = __int_as_float((__float_as_int(s) & 0x007FFFFF) | 0x3F800000);
    // the rounding of S to s goes in to first order
    return e * LN2 + (double)(logf(m) + (float)(S - (double)s) / s);
}

// The log-probability (-inf: no distribution, or none on the target), not
// above 0 by the terms' errors either.
__device__ __forceinline__ double row_logprob(const Args& a, const Row& w, float lt) {
    if (w.M == -INFINITY && w.S == 0.0) return -INFINITY;
    const double lp = ((double)lt * (double)a.k - w.R) * LN2 - ln_sum(w.S);
    return lp > 0.0 ? 0.0 : lp;
}

// The policy loss's derivative by the row's log-probability. F: the precision;
// a ratio at a border counts as not clipped, and an advantage of 0 takes
// nothing of an infinite ratio.
template <typename F>
__device__ __forceinline__ F policy_slope(F lo, F hi, F kl, F adv, F ratio, F eu, F* loss) {
    if (adv == (F)0 && ratio == ratio) ratio = (F)1;
    const F fit = ratio < lo ? lo : ratio > hi ? hi : ratio;  // NaN stays
    const F x = ratio * adv, y = fit * adv;
    *loss = x <= y ? -x : y < x ? -y : (F)NAN;
    return (x <= y ? -x : y < x ? (F)0 : (F)NAN) - (kl != (F)0 ? kl * eu : (F)0);
}

// e^d * f * ws, where e^d passes the fp32 range (d up to 176) and the product
// may not.
__device__ __forceinline__ float steep(float d, float f, float ws) {
    const float h = expf(0.5f * d);
    return h * ws * f * h;
}

// A row's gradient coefficients. All the row's threads wait for them, so the
// exponentials of differences of log-probabilities, which are near 1, are
// expf's here (2^-23 relative); their 64-bit forms took 1.4 us. Where ratio or
// KL factor passes fp32, slope and weight are multiplied by halves of it.
template <bool ENT>
__device__ __forceinline__ Coef row_coef(const Args& a, const Row& w, const RowIn& in) {
    const double lp = row_logprob(a, w, in.lt);
    const double d = lp - (double)in.old_lp, u = a.kl != 0.0 ? (double)in.ref_lp - lp : 0.0;
    const float S = (float)w.S, ratio = expf((float)d), eu = a.kl != 0.0 ? expm1f((float)u) : 0.0f;
    const float lo = (float)(1.0 - a.clip_lo), hi = (float)(1.0 + a.clip_hi), kl = (float)a.kl, ws = (float)(in.weight * a.scale);
    float loss, g = policy_slope<float>(lo, hi, kl, in.adv, ratio, eu, &loss) * ws;
    if (!finite(g) && d == d && u == u) {
        const bool out = in.adv == 0.0f || (in.adv > 0.0f ? ratio > hi : ratio < lo);
        g = ws == 0.0f ? 0.0f : (out ? 0.0f : -steep((float)d, in.adv, ws)) - (steep((float)u, kl, ws) - kl * ws);
    }
    Coef c = make_coef(w.M, (float)w.R, w.wide, S, ENT ? (float)-LN2 * ((float)w.Q / S) : 0.0f, g, ENT ? -(float)a.ec * ws : 0.0f, (float)a.inv_t);
    c.lt = target_logit(c, in.lt);
    return c;
}

// Writes a row's outputs (one thread of the calling warp). The loss is formed
// in 64 bits: a mean over rows of either sign keeps little of each.
template <bool ENT, bool POLICY>
__device__ __forceinline__ void write_row(const Args& a, int64_t r, const Row& w, const RowIn& in) {
    const bool none = w.M == -INFINITY && w.S == 0.0;
    const double lp = row_logprob(a, w, in.lt);
    double H = 0.0;
    if (ENT && !none) {
        const float S = (float)w.S, q = (float)w.Q / S;
        H = ln_sum(w.S) - LN2 * ((double)q + (double)((float)(w.Q - (double)q * w.S) / S));
        if (H < 0.0) H = 0.0;
    }
    a.logprob[r] = (float)lp;
    if (a.entropy) a.entropy[r] = (float)H;
    // S was summed against R, not M * k
    if (a.stats) a.stats[r] = {w.M, (float)(w.S * (none ? 1.0 : exp2(w.R - (double)w.M * (double)a.k)))};
    if (a.row_grad) a.row_grad[r] = 0.0f;
    if (POLICY) {
        const double u = a.kl != 0.0 ? (double)in.ref_lp - lp : 0.0, eu = a.kl != 0.0 ? expm1(u) : 0.0;
        double loss;
        policy_slope<double>(1.0 - a.clip_lo, 1.0 + a.clip_hi, a.kl, in.adv, exp(lp - (double)in.old_lp), eu, &loss);
        if (a.kl != 0.0) loss += a.kl * (isinf(eu) ? eu : eu - u);
        if (ENT && a.ec != 0.0) loss -= a.ec * H;
        a.row_loss[r] = (float)loss;
    }
}

// Outputs of a row that takes no part (0) or whose target is out of range (NaN).
template <bool POLICY>
__device__ __forceinline__ void blank_row(const Args& a, int64_t r, float v) {
    a.logprob[r] = v;
    if (a.entropy) a.entropy[r] = v;
    if (a.stats) a.stats[r] = {0.0f, 0.0f};
    if (a.row_grad) a.row_grad[r] = 0.0f;
    if (POLICY) a.row_loss[r] = v;
}

// ---- the gradient ------------------------------------------------------------

template <bool ENT>
__device__ __forceinline__ float grad1(const Coef& c, float l, float k) {
    const float t = c.kind == ROW_WIDE ? (l - c.c) * k : fmaf(l, k, -c.c);
    const float e = ex2_approx(t), f = ENT ? fmaf(c.b, fmaxf(t, -200.0f), c.a) : c.a;
    return c.kind == ROW_WIDE && e == 0.0f ? 0.0f : e * f;
}

// A pack's gradient (rows of ROW_SUM).
template <bool ENT, int N>
__device__ __forceinline__ void grad_pack(float (&x)[N], const Coef& c, float k) {
    const f32x2 nc = pack2(-c.c, -c.c), kk = pack2(k, k), aa = pack2(c.a, c.a), bb = pack2(c.b, c.b);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const f32x2 t = fma2(pack2(x[i], x[i + 1]), kk, nc);
        float t0, t1;
        unpack2(t, t0, t1);
        f32x2 e = pack2(ex2_approx(t0), ex2_approx(t1));
        e = mul2(e, ENT ? fma2(bb, pack2(fmaxf(t0, -200.0f), fmaxf(t1, -200.0f)), aa) : aa);
        unpack2(e, x[i], x[i + 1]);
    }
}

template <typename T, bool ENT>
__device__ __forceinline__ uint4 grad_of(const uint4& p, const Coef& c, float k) {
    float x[Type<T>::N];
    widen(p, x, (T*)nullptr);
    grad_pack<ENT>(x, c, k);
    return narrow(x, (T*)nullptr);
}

// The same for rows of ROW_WIDE (rare: out of the streaming loops).
template <typename T, bool ENT>
__device__ __noinline__ uint4 grad_of_wide(uint4 p, Coef c, float k) {
    float x[Type<T>::N];
    widen(p, x, (T*)nullptr);
#pragma unroll
    for (int i = 0; i < Type<T>::N; i++) x[i] = grad1<ENT>(c, x[i], k);
    return narrow(x, (T*)nullptr);
}

__device__ __forceinline__ bool elementwise(const Coef& c) { return c.kind == ROW_SUM || c.kind == ROW_WIDE; }

// A pack of zeros, or of NaN.
template <typename T>
__device__ __forceinline__ uint4 fill_pack(const Coef& c) {
    float x[Type<T>::N];
#pragma unroll
    for (int i = 0; i < Type<T>::N; i++) x[i] = c.kind == ROW_NAN ? NAN : 0.0f;
    return narrow(x, (T*)nullptr);
}

// Stores a pack whose place is not 16-byte aligned.
template <typename T>
__device__ __noinline__ void store_elements(T* dst, uint4 p) {
    const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (sizeof(T) == 4) {
            reinterpret_cast<uint32_t*>(dst)[i] = w[i];
        } else {
            reinterpret_cast<uint16_t*>(dst)[2 * i] = (uint16_t)w[i];
            reinterpret_cast<uint16_t*>(dst)[2 * i + 1] = (uint16_t)(w[i] >> 16);
        }
    }
}

// An edge element's gradient.
template <typename T, bool ENT>
__device__ __forceinline__ void put_edge(T* out, int v, int target, float l, const Coef& c, float k) {
    const bool hot = v == target;
    put1(out + v, c.kind == ROW_ZERO ? 0.0f : c.kind == ROW_NAN ? NAN : grad1<ENT>(c, hot ? target_logit(c, l) : l, k) + (hot ? c.one : 0.0f));
}

// Writes a row's gradient where no batch loop fits: element-wise gradients of
// wide rows, fills, and rows of another 16-byte phase than the logits'.
// Packs [lo, hi), pack lo + i by thread i % nt.
template <typename T, bool ENT>
__device__ __noinline__ void grad_plain(const T* row, T* out, int head, int lo, int hi, Coef c, float k, int tid, int nt) {
    const uint4* src = reinterpret_cast<const uint4*>(row + head);
    T* dst = out + head;
    const bool same = ((uintptr_t)dst & 15) == 0;
    const uint4 fill = fill_pack<T>(c);
#pragma unroll 4
    for (int v = lo + tid; v < hi; v += nt) {
        uint4 g = fill;
        if (elementwise(c)) {
            const uint4 p = load_pack(src + v);
            g = c.kind == ROW_SUM ? grad_of<T, ENT>(p, c, k) : grad_of_wide<T, ENT>(p, c, k);
        }
        if (same)
            reinterpret_cast<uint4*>(dst)[v] = g;
        else
            store_elements(dst + (int64_t)v * Type<T>::N, g);
    }
}

// ---- clusters ----------------------------------------------------------------

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void remote_store(uint32_t addr, int x) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(x) : "memory"); }
__device__ __forceinline__ void remote_store(uint32_t addr, const Part& p) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "f"(p.m), "f"(p.s), "f"(p.q), "f"(p.tag) : "memory");
}

// Sums of one thread's share of a slice against M itself, with differences
// taken before the multiply: for rows whose maximum is so large, or so low,
// that l * k - R would keep nothing of t (a row masked throughout). Such rows
// hold many equal terms, whose roundings share a sign: the sums of each 32 of
// them are added with the rounding errors carried on.
// UN: loads in flight; the per-row policy kernel, short of registers, spills
// more of its short rows' for the sake of 4 (20000 f16 rows of 1000 columns 42.1
// us against 40.0 with 2; 300 wide fp32 rows of 9001 20.0 and 20.1).
template <typename T, bool ENT, int UN>
__device__ __noinline__ Part wide_part(const T* row, int V, float M, float k, int part, int parts, int first, int nt) {
    const Slice sl = slice_of(row, V, part, parts, 0);
    const int v0 = part == 0 ? 0 : sl.head + sl.lo * Type<T>::N, v1 = part == parts - 1 ? V : sl.head + (sl.lo + sl.n) * Type<T>::N;
    float s = 0.0f, q = 0.0f, s_off = 0.0f, q_off = 0.0f;
    const auto carry = [](float& sum, float& off, float x) {
        const float y = x - off, z = sum + y;
        off = (z - sum) - y;
        sum = z;
    };
    for (int v = v0 + first; v < v1;) {
        float ps = 0.0f, pq = 0.0f;
        const int end = v1 - v > 32 * nt ? v + 32 * nt : v1;
#pragma unroll UN
        for (; v < end; v += nt) {
            const float t = (widen1(row[v]) - M) * k;
            const float e = ex2_approx(t);
            ps += e;
            if (ENT) pq = fmaf(e, fmaxf(t, -200.0f), pq);
        }
        carry(s, s_off, ps);
        if (ENT) carry(q, q_off, pq);
    }
    return Part{M, warp_sum(s), ENT ? warp_sum(q) : 0.0f, 0.0f};
}

// Joins such parts.
__device__ __forceinline__ Row join_wide(const Part* parts, int n, float M, float k) {
    const int lane = threadIdx.x & 31;
    Row w;
    double s = 0.0, q = 0.0;
    for (int i = lane; i < n; i += 32) s += (double)parts[i].s, q += (double)parts[i].q;
    w.M = M;
    w.S = warp_sum(s), w.Q = warp_sum(q);
    w.R = (double)M * (double)k;
    w.wide = true;
    return w;
}

// Lets a kernel launched behind this one with programmatic serialization start
// (it waits for this one's end before it reads).
__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---- a cluster per row ---------------------------------------------------------

// Log-probabilities, and the policy loss of few or of short rows: one cluster
// (or one CTA) per row, each CTA a slice of it. The sums come from memory; for
// the gradient the slice is read again, from L2 (or not at all: the last
// batch of packs is still in registers, which is all of a short slice).
// Measured at V = 151936: 8191 bf16 rows, a tenth of them left out, in 313 us
// (1.09 of the measured copy rate: reads are faster than copies); one fp32
// row in 4.4 us.
// With ROWS > 1 (NT = 32) a CTA's warps take a row each: short rows by CTAs of
// their own are bound by the rate at which CTAs start (20000 f16
// rows of 1000 columns: 53.8 us with a CTA of 128 threads a row, 16.0 with 8 rows
// a CTA).
template <typename T, bool ENT, bool POLICY, int NT, int ROWS>
__global__ void __launch_bounds__(NT * ROWS, 1024 / (NT * ROWS)) rows_kernel(const Args a) {
    static_assert(ROWS == 1 || NT == 32, "a row for each warp, or the CTA's threads for one row");
    constexpr int N = Type<T>::N, NW = NT / 32, STEP = NT * U;
    __shared__ Part parts_of[ROWS][2][MAXC * NW];
    __shared__ Coef coef_of[ROWS];
    __shared__ bool again_of[ROWS];
    __shared__ float wide_m_of[ROWS];
    const int C = ROWS == 1 ? (int)cluster_size() : 1, rank = ROWS == 1 ? (int)cluster_rank() : 0;
    const int group = ROWS == 1 ? 0 : (int)threadIdx.x / NT;
    const int tid = ROWS == 1 ? (int)threadIdx.x : (int)threadIdx.x % NT, lane = tid & 31, warp = tid >> 5;
    const int64_t r = ROWS == 1 ? (int64_t)(blockIdx.x / C) : (int64_t)blockIdx.x * ROWS + group;
    if (ROWS > 1 && r >= a.rows) {
        launch_next();
        return;
    }
    Part(&parts)[2][MAXC * NW] = parts_of[group];
    Coef& coef = coef_of[group];
    bool& again = again_of[group];
    float& wide_m = wide_m_of[group];
    const auto sync = [] {
        if (ROWS == 1)
            __syncthreads();
        else
            __syncwarp();
    };
    const T* row = (const T*)a.logits + r * a.ld;
    const float k = a.k;
    const int target = a.targets[r];
    const double weight = POLICY ? (a.weight ? (double)a.weight[r] : a.mean) : 1.0;
    const Slice s = slice_of(row, a.V, rank, C, tid);
    const uint4* src = reinterpret_cast<const uint4*>(row + s.head) + s.lo + tid;
    // the first batch is the ragged one, and on its way before the row is known to take part
    int first = s.n % STEP;
    if (first == 0) first = min(s.n, STEP);
    uint4 p[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        p[u] = make_uint4(Type<T>::NEG_INF, Type<T>::NEG_INF, Type<T>::NEG_INF, Type<T>::NEG_INF);
        if (u * NT + tid < first) p[u] = load_pack(src + u * NT);
    }
    if (C > 1) cluster_arrive();  // the peers' shared memory is written below

    const bool live = target >= 0 && weight != 0.0, bad = target >= a.V;
    T* out = (T*)a.grad + r * a.grad_ld;
    if (!live || bad) {
        if (C > 1) cluster_wait();
        launch_next();
        if (rank == 0 && tid == 0) blank_row<POLICY>(a, r, live ? NAN : 0.0f);
        if (POLICY && a.grad) {
            const Coef c = fill_coef(live);
            if (s.edge >= 0) put_edge<T, ENT>(out, s.edge, target, 0.0f, c, k);
            grad_plain<T, ENT>(row, out, s.head, s.lo, s.lo + s.n, c, k, tid, NT);
        }
        return;
    }
    RowIn in{0.0f, 0.0f, 0.0f, 0.0f, weight};
    if (warp == 0) {
        in.lt = widen1(row[target]);
        if (POLICY) {
            in.adv = a.adv[r], in.old_lp = a.old_lp[r];
            if (a.kl != 0.0) in.ref_lp = a.ref_lp[r];
        }
    }
    const float edge = s.edge >= 0 ? widen1(row[s.edge]) : -INFINITY;
    Acc acc = acc_new();
    int held = 0;  // the batch in p
    for (int v = first; v < s.n; v += STEP) {
        acc_packs<T, ENT>(acc, p, k);
#pragma unroll
        for (int u = 0; u < U; u++) p[u] = load_pack(src + v + u * NT);
        held = v;
    }
    acc_packs<T, ENT>(acc, p, k);
    if (s.edge >= 0) acc_one<ENT>(acc, edge, k);
    Part mine = warp_part<ENT>(acc, k);
    Row w{};            // warp 0: the row's sums
    float wide = 0.0f;  // M of a wide row in its second turn
    for (int turn = 0; turn < 2; turn++) {
        if (C > 1) {
            if (turn == 0) cluster_wait();  // the peers run
            if (lane < C) remote_store(map_rank(smem_u32(&parts[turn][rank * NW + warp]), lane), mine);
            cluster_arrive();
            cluster_wait();
        } else {
            if (lane == 0) parts[turn][warp] = mine;
            sync();
        }
        if (warp == 0) {
            w = turn ? join_wide(parts[1], C * NW, wide, k) : join_parts<ENT>(parts[0], C * NW, k);
            if (POLICY && a.grad && (turn || !w.wide)) {
                const Coef c = row_coef<ENT>(a, w, in);
                if (lane == 0) coef = c;
            }
            if (lane == 0) again = !turn && w.wide, wide_m = w.M;
        }
        sync();
        if (!again) break;
        wide = wide_m;
        mine = wide_part<T, ENT, POLICY ? 2 : 4>(row, a.V, wide, k, rank, C, tid, NT);
        sync();  // again and wide_m are written once more
    }
    if (rank == 0 && tid == 0) write_row<ENT, POLICY>(a, r, w, in);
    launch_next();
    if (!POLICY || !a.grad) return;

    const Coef c = coef;
    if (s.edge >= 0) put_edge<T, ENT>(out, s.edge, target, edge, c, k);
    T* dst = out + s.head + (int64_t)(s.lo + tid) * N;
    const int hot = target >= s.head ? (target - s.head) / N - s.lo : -1;  // the target's pack, if 0 <= hot < s.n
    int hot_thread = hot % NT;
    if (((uintptr_t)dst & 15) == 0 && c.kind == ROW_SUM) {
        uint4* d = reinterpret_cast<uint4*>(dst);
        const int end = held ? s.n : first;
#pragma unroll
        for (int u = 0; u < U; u++)
            if (held + u * NT + tid < end) __stcs(d + held + u * NT, (grad_of<T, ENT>(p[u], c, k)));
        for (int v = held - STEP; v >= first; v -= STEP) {
#pragma unroll
            for (int u = 0; u < U; u++) p[u] = load_pack(src + v + u * NT);
#pragma unroll
            for (int u = 0; u < U; u++) __stcs(d + v + u * NT, (grad_of<T, ENT>(p[u], c, k)));
        }
        if (held) {
#pragma unroll
            for (int u = 0; u < U; u++)
                if (u * NT + tid < first) p[u] = load_pack(src + u * NT);
#pragma unroll
            for (int u = 0; u < U; u++)
                if (u * NT + tid < first) __stcs(d + u * NT, (grad_of<T, ENT>(p[u], c, k)));
        }
        if (hot >= first) hot_thread = (hot - first) % NT;  // batches begin at first + i * STEP
    } else {
        grad_plain<T, ENT>(row, out, s.head, s.lo, s.lo + s.n, c, k, tid, NT);
    }
    // the thread that wrote the target's pack puts the target right
    if (hot >= 0 && hot < s.n && tid == hot_thread && elementwise(c)) put1(out + target, grad1<ENT>(c, c.lt, k) + c.one);
}

// ---- a stream of rows per cluster ----------------------------------------------

// The policy loss with its gradient over many long rows. Persistent clusters,
// each CTA a slice of every row of its cluster; a producer warp streams the
// slices through a ring of chunks in shared memory (bulk copies), a joining
// warp turns sums into coefficients, and NT consumer threads work on chunks in
// this order, the same in producer and consumers: chunks of row i for its
// sums, and behind the first LAG_CHUNKS of them, in turn with the others, the
// chunks of the row before for its gradient, read again from L2. So a row's
// sums travel to the joining warp and back while the consumers are busy, and
// loads of one row stand beside stores of another.
//
// The rows in flight, two per cluster (the one summed and the one before), have
// to stay in L2 (126 MB) between their two readings. The launcher takes the
// cluster size that brings one row per cluster under STREAM_L2 bytes, so twice
// that in flight; with 8 CTAs a row, the most, rows above 1.8 MB pass it (18
// clusters of 4 MB rows: 75 MB, and twice that), and middle rows, a CTA each, are
// 296 of up to 128 KB (39 MB, and twice that).
// Rows that take no part are left out of the stream (a bit per row in shared
// memory), so that every cluster gets the same number of live rows, and are
// filled at the end.
constexpr int LAG_CHUNKS = 1;
constexpr int STREAM_ROWS = 16384;  // rows of one launch at most

template <int NT_, int CTAS_, int PP_, int STAGES_>
struct StreamShape {
    static constexpr int NT = NT_;          // consumer threads
    static constexpr int CTAS = CTAS_;      // CTAs per SM
    static constexpr int PP = PP_;          // packs of a thread per chunk
    static constexpr int STAGES = STAGES_;  // chunks of the ring
    static constexpr int NW = NT / 32, CHP = NT * PP, CH = CHP * 16;
};

template <typename Shape>
struct StreamShared {
    Part own[2][Shape::NW];   // of the rows in turn, from the CTA's warps
    Part parts[2][MAXC];      // ... and from the cluster's CTAs
    Part wide_parts[MAXC];
    int sent[MAXC], wide_sent[MAXC];  // how many of them each CTA has sent here, at the end
    uint64_t full[Shape::STAGES], empty[Shape::STAGES];
    uint64_t obar[2], xbar[2], cbar[2], wbar;  // own parts, parts, coefficients, wide parts are here
    Coef coef[2];
    int rows[8];              // the rows whose first chunks are out, in turn
    uint32_t live[STREAM_ROWS / 32], before[STREAM_ROWS / 32];  // rows that take part; their number before each word
    int nlive;
    int abort;
};

// Stores p at a peer's shared address; the peer's barrier counts the bytes.
__device__ __forceinline__ void send_part(uint32_t addr, uint32_t bar, const Part& p) {
    asm volatile(
        "st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1,%2,%3,%4}, [%5];" ::"r"(addr), "f"(p.m),
        "f"(p.s), "f"(p.q), "f"(p.tag), "r"(bar)
        : "memory");
}

// Waits for a phase of `bar`. After WAIT_CYCLES (or the self-test's limit), or once another wait of the
// CTA has given up, returns all the same: the sums that the CTA has not handed
// in come out NaN, and all its gradients.
__device__ __forceinline__ void stream_wait(uint32_t bar, uint32_t parity, volatile int* abort, uint32_t selftest) {
    if (mbar_try_wait(bar, parity)) return;
    const long long t0 = clock64(), limit = selftest ? 1ll << (selftest >> 24) : WAIT_CYCLES;
    while (!mbar_try_wait(bar, parity)) {
        if (*abort) return;
        if (clock64() - t0 > limit) {
            *abort = 1;
            return;
        }
    }
}

// Waits until the part with this tag has landed (0: none was sent).
__device__ __forceinline__ void wait_landed(const Part& p, int tag) {
    const volatile float* at = &p.tag;
    const long long t0 = clock64();
    while (tag > 0 && __float_as_int(*at) != tag)
        if (clock64() - t0 > WAIT_CYCLES) return;
}

__device__ __forceinline__ uint4 lds_pack(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar, uint64_t pol) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(dst),
        "l"(src), "r"(bytes), "r"(bar), "l"(pol)
        : "memory");
}

// The j-th row (from 0) that takes part, or with dead that does not.
template <typename Shape>
__device__ __forceinline__ int64_t nth_row(const StreamShared<Shape>& sh, int rows, int j, bool dead) {
    int lo = 0, hi = (rows + 31) / 32;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2, n = (int)sh.before[mid];
        if ((dead ? 32 * mid - n : n) <= j)
            lo = mid;
        else
            hi = mid;
    }
    uint32_t m = dead ? ~sh.live[lo] : sh.live[lo];
    j -= dead ? 32 * lo - (int)sh.before[lo] : (int)sh.before[lo];
    for (; j > 0; j--) m &= m - 1;
    return 32 * lo + __ffs(m) - 1;
}

template <typename T, bool ENT, typename Shape>
__global__ void __launch_bounds__(Shape::NT + 64, Shape::CTAS) stream_kernel(const Args a) {
    constexpr int N = Type<T>::N, NT = Shape::NT, NW = Shape::NW, PP = Shape::PP, CHP = Shape::CHP, CH = Shape::CH;
    constexpr uint32_t STAGES = Shape::STAGES;
    extern __shared__ __align__(128) unsigned char ring[];
    __shared__ StreamShared<Shape> sh;
    const int C = (int)cluster_size(), rank = (int)cluster_rank();
    const int cid = (int)(blockIdx.x / C), step = (int)(gridDim.x / C);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t ring_u = smem_u32(ring), full_u = smem_u32(sh.full), empty_u = smem_u32(sh.empty);
    const uint32_t obar_u = smem_u32(sh.obar), xbar_u = smem_u32(sh.xbar), cbar_u = smem_u32(sh.cbar), wbar_u = smem_u32(&sh.wbar);
    volatile int* abort = &sh.abort;
    const float k = a.k;

    if (tid == 0) {
        for (uint32_t i = 0; i < STAGES; i++) {
            mbar_init(full_u + 8 * i, 1);
            mbar_init(empty_u + 8 * i, NW);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(obar_u + 8 * i, NW);
            mbar_init(xbar_u + 8 * i, 1);
            mbar_init(cbar_u + 8 * i, 1);
        }
        mbar_init(wbar_u, 1);
        for (int i = 0; i < MAXC; i++) sh.parts[0][i].tag = sh.parts[1][i].tag = sh.wide_parts[i].tag = 0.0f;
        sh.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    const int words = (a.rows + 31) / 32;
    for (int w = warp; w < words; w += NW + 2) {
        const int r = 32 * w + lane, t = r < a.rows ? a.targets[r] : -1;
        const unsigned m = __ballot_sync(FULL, t >= 0 && t < a.V && !(a.weight && a.weight[r] == 0.0f));
        if (lane == 0) sh.live[w] = m;
    }
    __syncthreads();
    if (warp == 0) {
        int sum = 0;
        for (int w0 = 0; w0 < words; w0 += 32) {
            const int n = w0 + lane < words ? __popc(sh.live[w0 + lane]) : 0, upto = warp_incl_scan(n, lane);
            if (w0 + lane < words) sh.before[w0 + lane] = (uint32_t)(sum + upto - n);
            sum += __shfl_sync(FULL, upto, 31);
        }
        if (lane == 0) sh.nlive = sum;
    }
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    const int mine_n = sh.nlive > cid ? (sh.nlive - cid + step - 1) / step : 0;  // rows of this cluster

    if (warp == NW) {  // ---- the producer warp: its first lane issues the copies
        if (lane == 0) {
            uint64_t again, once;
            asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(again));
            asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(once));
            uint32_t stage = 0, phase = 0, issued = 0;
            const uint32_t stop = a.selftest && cid == 0 && rank == C - 1 ? (a.selftest & 0xFFFFFFu) - 1 : ~0u;
            const uint4* b_src = nullptr;  // the row before, whose gradient is due
            int b_n = 0, b_packs = 0;
            const auto put = [&](const uint4* src, int j, int packs, uint64_t pol) {
                const uint32_t bytes = (uint32_t)min(CHP, packs - j * CHP) * 16;
                if (issued == stop) return;
                stream_wait(empty_u + 8 * stage, phase ^ 1, abort, a.selftest);
                if (*abort) return;
                mbar_arrive_tx(full_u + 8 * stage, bytes);
                bulk_load(ring_u + stage * CH, src + j * CHP, bytes, full_u + 8 * stage, pol);
                issued++;
                if (++stage == STAGES) stage = 0, phase ^= 1;
            };
            for (int i = 0; i <= mine_n && !*abort; i++) {
                const uint4* src = nullptr;
                int n = 0, packs = 0;
                if (i < mine_n) {
                    const int64_t r = nth_row(sh, a.rows, cid + i * step, false);
                    const T* row = (const T*)a.logits + r * a.ld;
                    const Slice s = slice_of(row, a.V, rank, C, tid);
                    src = reinterpret_cast<const uint4*>(row + s.head) + s.lo;
                    packs = s.n, n = (s.n + CHP - 1) / CHP;
                    sh.rows[i & 7] = (int)r;
                }
                const int lag = min(n, LAG_CHUNKS), steps = max(n, lag + b_n);
                for (int j = 0; j < steps && !*abort; j++) {
                    if (j < n) put(src, j, packs, again);
                    if (j >= lag && j - lag < b_n) put(b_src, j - lag, b_packs, once);
                }
                b_src = src, b_n = n, b_packs = packs;
            }
            // the copies in flight land before the CTA leaves, whoever has given up
            const uint32_t n = min(issued, STAGES);
            for (uint32_t i = 0; i < n; i++) {
                if (stage == 0) stage = STAGES, phase ^= 1;
                stage--;
                mbar_wait(full_u + 8 * stage, phase);
            }
        }
    } else if (warp == NW + 1) {  // ---- the joining warp: sums to coefficients
        uint32_t phases = 0;  // of xbar and obar, a bit for each parity
        uint32_t wphase = 0;
        int sent = 0, wide_sent = 0;  // parts that this lane has sent to its peer, each with its number as tag
        const auto inputs = [&](int64_t r) {
            RowIn in{0.0f, 0.0f, 0.0f, 0.0f, 0.0};
            in.lt = widen1(((const T*)a.logits + r * a.ld)[a.targets[r]]);
            in.adv = a.adv[r], in.old_lp = a.old_lp[r];
            if (a.kl != 0.0) in.ref_lp = a.ref_lp[r];
            in.weight = a.weight ? (double)a.weight[r] : a.mean;
            return in;
        };
        int64_t next = mine_n ? nth_row(sh, a.rows, cid, false) : 0;
        RowIn next_in = mine_n ? inputs(next) : RowIn{};
        for (int i = 0; i < mine_n; i++) {
            const int par = i & 1;
            const int64_t r = next;
            const RowIn in = next_in;
            // the next row's target is read before this row's coefficients are
            // out: behind them a peer may come to write over the next row
            if (i + 1 < mine_n) {
                next = nth_row(sh, a.rows, cid + (i + 1) * step, false);
                next_in = inputs(next);
            }
            stream_wait(obar_u + 8 * par, (phases >> par) & 1, abort, a.selftest);
            const bool gone = *abort;  // nothing is sent, and no barrier armed again, once a wait has given up
            Row w = join_parts<ENT>(sh.own[par], NW, k);
            if (C > 1) {
                if (lane == 0 && !gone) mbar_arrive_tx(xbar_u + 8 * par, C * 16);
                __syncwarp();
                if (lane < C && !gone) {
                    sent = i + 1;
                    send_part(map_rank(smem_u32(&sh.parts[par][rank]), lane), map_rank(xbar_u + 8 * par, lane),
                              Part{w.M, (float)w.S, (float)w.Q, __int_as_float(sent)});
                }
                stream_wait(xbar_u + 8 * par, (phases >> par) & 1, abort, a.selftest);
                w = join_parts<ENT>(sh.parts[par], C, k);
            }
            phases ^= 1u << par;
            if (*abort) w.S = NAN, w.wide = false;
            if (w.wide) {  // the same in every CTA: once more through the slices, by these warps
                const T* row = (const T*)a.logits + r * a.ld;
                Part own = wide_part<T, ENT, 4>(row, a.V, w.M, k, rank, C, lane, 32);
                if (lane == 0 && !*abort) mbar_arrive_tx(wbar_u, C * 16);
                __syncwarp();
                if (lane < C && !*abort) {
                    own.tag = __int_as_float(++wide_sent);
                    send_part(map_rank(smem_u32(&sh.wide_parts[rank]), lane), map_rank(wbar_u, lane), own);
                }
                stream_wait(wbar_u, wphase, abort, a.selftest);
                wphase ^= 1;
                w = join_wide(sh.wide_parts, C, w.M, k);
                if (*abort) w.S = NAN;
            }
            const Coef c = row_coef<ENT>(a, w, in);
            if (lane == 0) {
                sh.coef[par] = c;
                mbar_arrive(cbar_u + 8 * par);
                if (rank == 0) write_row<ENT, true>(a, r, w, in);
            }
            __syncwarp();
        }
        if (C > 1 && lane < C) {
            remote_store(map_rank(smem_u32(&sh.sent[rank]), lane), sent);
            remote_store(map_rank(smem_u32(&sh.wide_sent[rank]), lane), wide_sent);
        }
    } else {  // ---- the consumers
        uint32_t stage = 0, phase = 0, cphase = 0;
        // the row before, whose gradient is due
        T* b_out = nullptr;
        Slice b{};
        int b_n = 0;
        float b_edge = 0.0f;
        int b_target = -1;
        for (int i = 0; i <= mine_n; i++) {
            const int par = i & 1;
            const bool more = i < mine_n;
            Slice s{};
            s.edge = -1;
            const T* row = nullptr;
            int64_t r = 0;
            float edge = -INFINITY;
            int n = 0;
            if (more) {  // the row's number comes with its first chunk
                stream_wait(full_u + 8 * stage, phase, abort, a.selftest);
                r = *abort ? nth_row(sh, a.rows, cid + i * step, false) : *(volatile int*)&sh.rows[i & 7];
                row = (const T*)a.logits + r * a.ld;
                s = slice_of(row, a.V, rank, C, tid);
                n = (s.n + CHP - 1) / CHP;
                if (s.edge >= 0) edge = widen1(row[s.edge]);
            }
            const int lag = min(n, LAG_CHUNKS), steps = max(more ? n + 1 : 0, lag + b_n);
            Acc acc = acc_new();
            Coef c;
            bool have_c = i == 0;
            T* b_dst = b_out + b.head + (int64_t)b.lo * N;
            const bool same = ((uintptr_t)b_dst & 15) == 0;
            const auto want_c = [&]() {  // the coefficients of the row before
                if (have_c) return;
                stream_wait(cbar_u + 8 * (par ^ 1), (cphase >> (par ^ 1)) & 1, abort, a.selftest);
                cphase ^= 1u << (par ^ 1);
                c = sh.coef[par ^ 1];
                have_c = true;
            };
            for (int j = 0; j < steps; j++) {
                if (j < n) {
                    stream_wait(full_u + 8 * stage, phase, abort, a.selftest);
                    const uint32_t at = ring_u + stage * CH + tid * 16;
                    uint4 p[PP];
                    if (j + 1 < n) {
#pragma unroll
                        for (int u = 0; u < PP; u++) p[u] = lds_pack(at + u * NT * 16);
                    } else {
#pragma unroll
                        for (int u = 0; u < PP; u++) {
                            p[u] = make_uint4(Type<T>::NEG_INF, Type<T>::NEG_INF, Type<T>::NEG_INF, Type<T>::NEG_INF);
                            if (j * CHP + u * NT + tid < s.n) p[u] = lds_pack(at + u * NT * 16);
                        }
                    }
                    acc_packs<T, ENT>(acc, p, k);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(empty_u + 8 * stage);
                    if (++stage == STAGES) stage = 0, phase ^= 1;
                } else if (j == n && more) {
                    if (s.edge >= 0) acc_one<ENT>(acc, edge, k);
                    const Part mine = warp_part<ENT>(acc, k);
                    // two buffers in turn: a warp hands in row i + 1 only with row i's coefficients in hand
                    want_c();
                    if (lane == 0) {
                        sh.own[par][warp] = mine;
                        mbar_arrive(obar_u + 8 * par);
                    }
                    __syncwarp();
                }
                if (j >= lag && j - lag < b_n) {
                    want_c();
                    const int base = (j - lag) * CHP + tid;
                    stream_wait(full_u + 8 * stage, phase, abort, a.selftest);
                    const uint32_t at = ring_u + stage * CH + tid * 16;
                    uint4* d = reinterpret_cast<uint4*>(b_dst) + base;
                    if (same && c.kind == ROW_SUM && j - lag + 1 < b_n) {
#pragma unroll
                        for (int u = 0; u < PP; u++) __stcs(d + u * NT, (grad_of<T, ENT>(lds_pack(at + u * NT * 16), c, k)));
                    } else {
#pragma unroll 1
                        for (int u = 0; u < PP; u++)
                            if (base + u * NT < b.n) {
                                const uint4 p = lds_pack(at + u * NT * 16);
                                const uint4 g = c.kind == ROW_SUM ? grad_of<T, ENT>(p, c, k) : c.kind == ROW_WIDE ? grad_of_wide<T, ENT>(p, c, k) : fill_pack<T>(c);
                                if (same)
                                    __stcs(d + u * NT, g);
                                else
                                    store_elements(b_dst + (int64_t)(base + u * NT) * N, g);
                            }
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(empty_u + 8 * stage);
                    if (++stage == STAGES) stage = 0, phase ^= 1;
                }
            }
            if (i > 0) {
                want_c();
                if (b.edge >= 0) put_edge<T, ENT>(b_out, b.edge, b_target, b_edge, c, k);
                // the thread that wrote the target's pack puts the target right
                const int hot = b_target >= b.head ? (b_target - b.head) / N - b.lo : -1;
                if (hot >= 0 && hot < b.n && hot % NT == tid && elementwise(c)) put1(b_out + b_target, grad1<ENT>(c, c.lt, k) + c.one);
            }
            if (more) {
                b_out = (T*)a.grad + r * a.grad_ld;
                b = s, b_n = n, b_edge = edge, b_target = a.targets[r];
            }
        }
        const auto fill = [&](int64_t r, int part, int parts, bool nan) {
            const T* row = (const T*)a.logits + r * a.ld;
            T* out = (T*)a.grad + r * a.grad_ld;
            const Slice s = slice_of(row, a.V, part, parts, tid);
            const Coef c = fill_coef(nan);
            if (s.edge >= 0) put_edge<T, ENT>(out, s.edge, -1, 0.0f, c, k);
            grad_plain<T, ENT>(row, out, s.head, s.lo, s.lo + s.n, c, k, tid, NT);
        };
        // a thread whose wait gave up has written what the ring held: NaN over all that it has written
        if (*abort)
            for (int i = 0; i < mine_n; i++) fill(nth_row(sh, a.rows, cid + i * step, false), rank, C, true);
        // rows that take no part: zeros, or NaN for a target out of range
        for (int j = (int)blockIdx.x; j < a.rows - sh.nlive; j += (int)gridDim.x) {
            const int64_t r = nth_row(sh, a.rows, j, true);
            const bool nan = a.targets[r] >= a.V && !(a.weight && a.weight[r] == 0.0f);
            if (tid == 0) blank_row<true>(a, r, nan ? NAN : 0.0f);
            fill(r, 0, 1, nan);
        }
    }
    // no CTA leaves while a peer may still store into its shared memory, or
    // while a part is on its way to it: those of rows that it has joined have
    // landed, and where its waits gave up, the last two rows' may not have
    __syncwarp();
    launch_next();
    cluster_arrive();
    cluster_wait();
    if (*abort && C > 1 && warp == NW + 1 && lane < C) {
        const int n = sh.sent[lane];
        wait_landed(sh.parts[(n + 1) & 1][lane], n);
        wait_landed(sh.parts[n & 1][lane], n - 1);
        wait_landed(sh.wide_parts[lane], sh.wide_sent[lane]);
    }
}

// ---- the gradient from given sums -------------------------------------------------

// One CTA per slice of a row, `parts` of them in turn: one read and one write.
// Measured: 2047 bf16 rows of 151936, a fifth of them zeros, in 178 us (0.96
// of the measured copy rate) with slices of 76 KB; slices of a quarter of
// that, in which a CTA's start weighs more, take 182 us.
// ROWS > 1: a warp for each row, for short ones (20000 f16 rows of 1000
// columns: 60 us with a CTA for each, 20 with a warp).
template <typename T, bool ENT, int ROWS>
__global__ void __launch_bounds__(256, 6) grad_kernel(const Args a, const int parts) {
    constexpr int N = Type<T>::N, NT = 256 / ROWS;
    wait_before();
    const int tid = ROWS == 1 ? (int)threadIdx.x : (int)threadIdx.x % NT;
    const int64_t r = ROWS == 1 ? (int64_t)(blockIdx.x / (unsigned)parts) : (int64_t)blockIdx.x * ROWS + threadIdx.x / NT;
    if (ROWS > 1 && r >= a.rows) return;
    const int part = ROWS == 1 ? (int)(blockIdx.x - (unsigned)r * (unsigned)parts) : 0;
    const float k = a.k;
    const int target = a.targets[r];
    const float g_lp = a.g_lp[r], g_ent = ENT ? a.g_ent[r] : 0.0f, ent = ENT ? a.ent_in[r] : 0.0f;
    const quasar_logprob_stat st = a.stats_in[r];
    const T* row = (const T*)a.logits + r * a.ld;
    T* out = (T*)a.grad + r * a.grad_ld;
    const Slice s = slice_of(row, a.V, part, ROWS == 1 ? parts : 1, tid);
    Coef c = fill_coef(target >= a.V && !(a.row_grad && g_lp == 0.0f));
    if (target >= 0 && target < a.V) {
        const float R = rintf(st.max * k);
        const bool wide = !(fabsf(R) < WIDE) && !isinf(st.max);
        // st.sum stands against M * k, the loop's terms against R
        const float S = wide || isinf(st.max) ? st.sum : st.sum * exp2f(fmaf(st.max, k, -R));
        c = make_coef(st.max, R, wide, S, ENT ? ent - logf(S) : 0.0f, g_lp, g_ent, (float)a.inv_t);
    }
    const int hot = target >= s.head ? (target - s.head) / N - s.lo : -1;
    const bool mine = elementwise(c) && hot >= 0 && hot < s.n && hot % NT == tid;
    const float lt = mine ? widen1(row[target]) : 0.0f;  // read before its pack is written over
    if (s.edge >= 0) put_edge<T, ENT>(out, s.edge, target, elementwise(c) ? widen1(row[s.edge]) : 0.0f, c, k);
    const uint4* src = reinterpret_cast<const uint4*>(row + s.head) + s.lo + tid;
    T* dst = out + s.head + (int64_t)(s.lo + tid) * N;
    if (((uintptr_t)dst & 15) == 0 && c.kind == ROW_SUM) {
        uint4* d = reinterpret_cast<uint4*>(dst);
        const int n = s.n - tid;
        int v = 0;
        for (; v + (U - 1) * NT < n; v += NT * U) {
            uint4 p[U];
#pragma unroll
            for (int u = 0; u < U; u++) p[u] = load_pack(src + v + u * NT);
#pragma unroll
            for (int u = 0; u < U; u++) d[v + u * NT] = grad_of<T, ENT>(p[u], c, k);
        }
        uint4 p[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (v + u * NT < n) p[u] = load_pack(src + v + u * NT);
#pragma unroll
        for (int u = 0; u < U; u++)
            if (v + u * NT < n) d[v + u * NT] = grad_of<T, ENT>(p[u], c, k);
    } else {
        grad_plain<T, ENT>(row, out, s.head, s.lo, s.lo + s.n, c, k, tid, NT);
    }
    if (mine) put1(out + target, grad1<ENT>(c, target_logit(c, lt), k) + c.one);
}

// ---- pairs and sums --------------------------------------------------------------

// Sum over a CTA, the same in every run; all threads get it.
__device__ __forceinline__ double cta_sum(double x, double* buf, int threads) {
    x = warp_sum(x);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = x;
    __syncthreads();
    double s = 0.0;
    for (int i = 0; i < threads / 32; i++) s += buf[i];
    return s;
}

__device__ __forceinline__ double pair_weight(const PairArgs& p, int i) { return p.weight ? (double)p.weight[i] : 1.0 / p.pairs; }

// Pair i by a warp, or by the CTA's 128 threads: its outputs and its rows'
// derivatives. Returns its loss in 64 bits.
template <bool WARP>
__device__ __forceinline__ double pair_loss(const PairArgs& p, int i, int tid, double* buf) {
    constexpr int NT = WARP ? 32 : 128;
    const int at[3] = {p.cu[2 * i], p.cu[2 * i + 1], p.cu[2 * i + 2]};
    const bool ok = at[0] >= 0 && at[0] <= at[1] && at[1] <= at[2] && at[2] <= p.rows;
    // before the sums, whose barriers stand between these and the outputs: seq may be ref
    const double ref[2] = {p.ref ? (double)p.ref[2 * i] : 0.0, p.ref ? (double)p.ref[2 * i + 1] : 0.0};
    double sum[2] = {0.0, 0.0}, n[2] = {0.0, 0.0};
    if (ok) {
        for (int s = 0; s < 2; s++) {
            double x = 0.0, c = 0.0;
            for (int64_t r = (int64_t)at[s] + tid; r < at[s + 1]; r += NT)
                if (p.targets[r] >= 0) x += (double)p.logprob[r], c += 1.0;
            sum[s] = WARP ? warp_sum(x) : cta_sum(x, buf, NT);
            n[s] = WARP ? warp_sum(c) : cta_sum(c, buf, NT);
        }
    } else {
        sum[0] = sum[1] = NAN;
    }
    double score[2], by[2];
    for (int s = 0; s < 2; s++) {
        by[s] = p.mean && n[s] > 0.0 ? 1.0 / n[s] : 1.0;
        score[s] = sum[s] * by[s] - ref[s];
    }
    const double x = p.beta * (score[0] - score[1]);
    // softplus(-x) and softplus(x); sigmoid(-x) and sigmoid(x)
    const double tail = log1p(exp(-fabs(x)));
    const double up = fmax(-x, 0.0) + tail, down = fmax(x, 0.0) + tail;
    const double sn = 1.0 / (1.0 + exp(x)), sp = 1.0 / (1.0 + exp(-x));
    // a share of 0 takes nothing, of an infinite loss either
    const double loss = x != x ? NAN : (p.eps != 1.0 ? (1.0 - p.eps) * up : 0.0) + (p.eps != 0.0 ? p.eps * down : 0.0);
    const double w = pair_weight(p, i);
    const double g = w != 0.0 ? -p.beta * ((1.0 - p.eps) * sn - p.eps * sp) * w * p.scale : 0.0;
    if (tid == 0) {
        p.seq[2 * i] = (float)sum[0];
        p.seq[2 * i + 1] = (float)sum[1];
        p.pair_loss[i] = (float)loss;
    }
    if (ok)
        for (int s = 0; s < 2; s++)
            for (int64_t r = (int64_t)at[s] + tid; r < at[s + 1]; r += NT)
                if (p.targets[r] >= 0) p.row_grad[r] = (float)((s ? -g : g) * by[s]);
    return loss;
}

// One CTA per pair.
__global__ void __launch_bounds__(128) pair_kernel(const PairArgs p) {
    __shared__ double buf[4];
    wait_before();
    launch_next();
    pair_loss<false>(p, (int)blockIdx.x, (int)threadIdx.x, buf);
}

// A warp per pair, and their weighted sum: for the pairs of a small batch,
// where a launch weighs more than the longer loops.
constexpr int FEW_PAIRS = 16, FEW_ROWS = 512;
__global__ void __launch_bounds__(32 * FEW_PAIRS) few_pairs_kernel(const PairArgs p, float* out) {
    __shared__ double part[FEW_PAIRS];
    wait_before();
    launch_next();
    const int i = (int)threadIdx.x / 32;
    if (i < p.pairs) {
        const double loss = pair_loss<true>(p, i, (int)threadIdx.x % 32, nullptr), w = pair_weight(p, i);
        if (threadIdx.x % 32 == 0) part[i] = w != 0.0 ? w * loss : 0.0;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double s = 0.0;
        for (int j = 0; j < p.pairs; j++) s += part[j];
        out[0] = (float)s;
    }
}

// One CTA: the same order of sums in every run. A weight of 0 takes nothing,
// of an infinite x either.
__global__ void __launch_bounds__(1024) weighted_sum_kernel(const float* x, const float* w, int n, float* out) {
    __shared__ double buf[32];
    wait_before();
    launch_next();
    double s = 0.0;
#pragma unroll 8
    for (int64_t i = threadIdx.x; i < n; i += 1024) {
        const float wi = w ? w[i] : 1.0f, xi = x[i];
        s += wi != 0.0f ? (double)wi * (double)xi : 0.0;
    }
    s = cta_sum(s, buf, 1024);
    if (threadIdx.x == 0) out[0] = (float)(w || n == 0 ? s : s / n);
}

// ---- launchers ---------------------------------------------------------------

// Starts `kern` behind what is on the stream; with `early` before that has
// ended (the kernel waits for it itself), which hides the launch.
template <typename... P, typename... X>
static cudaError_t launch(void (*kern)(P...), unsigned grid, int block, size_t smem, int cluster, bool early, cudaStream_t st, X... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3((unsigned)block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    unsigned n = 0;
    if (cluster > 0) {
        at[n].id = cudaLaunchAttributeClusterDimension;
        at[n].val.clusterDim.x = (unsigned)cluster;
        at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
        n++;
    }
    if (early) {
        at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[n].val.programmaticStreamSerializationAllowed = 1;
        n++;
    }
    cfg.attrs = at;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

static constexpr int SMS = 148;

// CTAs per row: clusters of up to 8 while the rows alone leave SMs idle, and
// the slices are not under 8 KB. At V = 151936, fp32: 1 row 4.4 us with 8
// CTAs and 10.8 with one; 256 rows 26.7 us with 2, 30.6 with 1, 29.8 with 4.
static int row_cluster(int64_t rows, int64_t row_bytes) {
    int C = 1;
    while (C < MAXC && rows * C < 2 * SMS && row_bytes >= (int64_t)C * 2 * 8192) C *= 2;
    return C;
}

template <typename T, bool ENT, bool POLICY, int NT, int ROWS>
static cudaError_t rows_launch(const Args& a, int C, cudaStream_t st) {
    const unsigned grid = ((unsigned)a.rows + ROWS - 1) / ROWS * (unsigned)C;
    return launch(rows_kernel<T, ENT, POLICY, NT, ROWS>, grid, NT * ROWS, 0, ROWS == 1 ? C : 0, false, st, a);
}

// Rows that a warp takes alone, in bytes: 20000 bf16 rows of 4000 columns,
// policy loss and gradient, 78 us against 112 with 128 threads a row; 500 rows
// of 18 KB 17.4 against 11.4.
static constexpr int64_t ROW_SHORT = 8192;

// Short rows take small CTAs, of which an SM runs more at once: a CTA's start,
// its barrier and its scalars take about 4 us whatever its slice. bf16 rows of
// 38 KB, 16384 of them: 255 us with 128 threads, 274 with 256 (policy loss and
// gradient); fp32 rows of 76 KB, 2000 of them: 62 us with 256, 69 with 128.
template <typename T, bool ENT, bool POLICY>
static cudaError_t rows_by_size(const Args& a, cudaStream_t st) {
    const int64_t row_bytes = (int64_t)a.V * sizeof(T);
    const int C = row_cluster(a.rows, row_bytes);
    if (C == 1 && row_bytes <= ROW_SHORT) return rows_launch<T, ENT, POLICY, 32, 8>(a, C, st);
    if (C == 1 && row_bytes <= 49152) return rows_launch<T, ENT, POLICY, 128, 1>(a, C, st);
    return rows_launch<T, ENT, POLICY, 256, 1>(a, C, st);
}

// Long rows: one CTA of 640 consumers per SM with chunks of 30 KB, and of 448
// with chunks of 28 KB for the entropy of 16-bit types, which is bound by
// instructions and has 119 registers a thread instead of 80 (bf16, long runs:
// V = 200000, 1500 rows 251 us against 261; V = 100000, 3000 rows 253 and 258;
// about even at V = 151936, 2000 rows 268 and 264, 1023 rows with KL term 116 and
// 113). Without entropy the two are even (V = 200000, 216), and in fp32, bound by
// memory, 640 are faster (2000 rows with entropy 391 and 405).
// Middle rows, of which an SM can hold two: two CTAs of 256 with chunks of 20 KB.
template <typename T, bool ENT>
using StreamLong =
    std::conditional_t<ENT && sizeof(T) == 2, StreamShape<448, 1, 4, 7>, StreamShape<640, 1, 3, 7>>;
using StreamMiddle = StreamShape<256, 2, 5, 5>;
static constexpr int64_t STREAM_MIN = 96 * 1024, STREAM_MIDDLE = 128 * 1024, STREAM_L2 = 32 << 20;

static std::mutex g_mu;

template <typename T, bool ENT, typename Shape>
static cudaError_t stream_launch(const Args& a, int C, cudaStream_t st) {
    auto kern = stream_kernel<T, ENT, Shape>;
    const size_t smem = (size_t)Shape::STAGES * Shape::CH;
    // per device: whether the kernel is set up, and the clusters that fit
    static int most[64][MAXC + 1];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    int clusters;
    {
        std::lock_guard<std::mutex> lock(g_mu);
        clusters = most[dev][C];
        if (!clusters) {
            e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
            if (e != cudaSuccess) return e;
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3((unsigned)C);
            cfg.blockDim = dim3(Shape::NT + 64);
            cfg.dynamicSmemBytes = smem;
            cudaLaunchAttribute at[1];
            at[0].id = cudaLaunchAttributeClusterDimension;
            at[0].val.clusterDim.x = (unsigned)C;
            at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
            cfg.attrs = at;
            cfg.numAttrs = 1;
            e = cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg);
            if (e != cudaSuccess) return e;
            if (clusters < 1) return cudaErrorInvalidConfiguration;
            most[dev][C] = clusters;
        }
    }
    for (int64_t r0 = 0; r0 < a.rows; r0 += STREAM_ROWS) {
        Args b = a;
        b.rows = (int)(a.rows - r0 < STREAM_ROWS ? a.rows - r0 : STREAM_ROWS);
        b.logits = (const T*)a.logits + r0 * a.ld;
        b.grad = (T*)a.grad + r0 * a.grad_ld;
        b.targets += r0, b.logprob += r0, b.row_loss += r0, b.old_lp += r0, b.adv += r0;
        if (b.entropy) b.entropy += r0;
        if (b.ref_lp) b.ref_lp += r0;
        if (b.weight) b.weight += r0;
        const int n = b.rows < clusters ? b.rows : clusters;
        e = launch(kern, (unsigned)(n * C), Shape::NT + 64, smem, C, false, st, b);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

// The policy loss with its gradient: the streaming kernel where a row is long
// enough for its chunks and there are rows for several turns of every cluster
// (policy loss and gradient at V = 151936: fp32, 4096 rows 745 us streamed,
// 1040 with a CTA per row; bf16, 600 rows 79 to 87 and 102 us, 148 rows 28 to 29
// and 27; 50021 f16 columns, 3001 rows 118 and 131 us, 1000 rows 48 and 51, 300
// rows 25.7 and 21.8).
template <typename T, bool ENT>
static cudaError_t policy_by_size(const Args& a, cudaStream_t st) {
    const int64_t row_bytes = (int64_t)a.V * sizeof(T);
    if (row_bytes >= STREAM_MIN && row_bytes <= STREAM_MIDDLE && a.rows >= 4 * SMS) return stream_launch<T, ENT, StreamMiddle>(a, 1, st);
    if (row_bytes > STREAM_MIDDLE && a.rows >= SMS) {
        int C = 1;
        while (C < MAXC && SMS / C * row_bytes > STREAM_L2) C *= 2;
        return stream_launch<T, ENT, StreamLong<T, ENT>>(a, C, st);
    }
    return rows_by_size<T, ENT, true>(a, st);
}

template <typename T>
static cudaError_t rows_typed(const Args& a, cudaStream_t st) {
    const bool ent = a.entropy != nullptr || a.ec != 0.0;
    if (!a.adv) return ent ? rows_by_size<T, true, false>(a, st) : rows_by_size<T, false, false>(a, st);
    if (!a.grad) return ent ? rows_by_size<T, true, true>(a, st) : rows_by_size<T, false, true>(a, st);
    return ent ? policy_by_size<T, true>(a, st) : policy_by_size<T, false>(a, st);
}

cudaError_t launch_rows(const Args& a, int dtype, cudaStream_t st) {
    if (dtype == QUASAR_F32) return rows_typed<float>(a, st);
    if (dtype == QUASAR_F16) return rows_typed<__half>(a, st);
    return rows_typed<__nv_bfloat16>(a, st);
}

// Slices of about 76 KB, smaller ones where the rows are few.
template <typename T>
static cudaError_t grad_typed(const Args& a, cudaStream_t st) {
    const int64_t row_bytes = (int64_t)a.V * sizeof(T);
    if (row_bytes <= ROW_SHORT) {
        const unsigned grid = ((unsigned)a.rows + 7) / 8;
        if (a.g_ent) return launch(grad_kernel<T, true, 8>, grid, 256, 0, 0, true, st, a, 1);
        return launch(grad_kernel<T, false, 8>, grid, 256, 0, 0, true, st, a, 1);
    }
    int64_t parts = (row_bytes + 77823) / 77824;
    while (parts * a.rows < 4 * SMS && row_bytes > parts * 2 * 8192) parts *= 2;
    if (parts * a.rows > INT32_MAX) parts = 1;
    const unsigned grid = (unsigned)(a.rows * parts);
    if (a.g_ent) return launch(grad_kernel<T, true, 1>, grid, 256, 0, 0, true, st, a, (int)parts);
    return launch(grad_kernel<T, false, 1>, grid, 256, 0, 0, true, st, a, (int)parts);
}

cudaError_t launch_grad(const Args& a, int dtype, cudaStream_t st) {
    if (dtype == QUASAR_F32) return grad_typed<float>(a, st);
    if (dtype == QUASAR_F16) return grad_typed<__half>(a, st);
    return grad_typed<__nv_bfloat16>(a, st);
}

cudaError_t launch_pairs(const PairArgs& p, float* loss, cudaStream_t st) {
    if (p.pairs > 0 && p.pairs <= FEW_PAIRS && p.rows <= FEW_ROWS) return launch(few_pairs_kernel, 1u, 32 * FEW_PAIRS, 0, 0, true, st, p, loss);
    if (p.pairs > 0) {
        const cudaError_t e = launch(pair_kernel, (unsigned)p.pairs, 128, 0, 0, true, st, p);
        if (e != cudaSuccess) return e;
    }
    return launch_weighted_sum(p.pair_loss, p.weight, p.pairs, loss, st);
}

cudaError_t launch_weighted_sum(const float* x, const float* w, int n, float* out, cudaStream_t st) {
    return launch(weighted_sum_kernel, 1u, 1024, 0, 0, true, st, x, w, n, out);
}

}  // namespace loss
}  // namespace qs
