// token_loss.cu - kernels of the token log-probabilities and of the losses
// made of them (include/quasar_losses.h).
//
// The mathematics: with M the largest logit of a row and d = l - M, the row's
// softmax needs S = sum 2^(d*k), k = log2(e)/T, and its entropy also
// Q = sum 2^(d*k) * d*k:  logprob = ln2 * (d_target*k - log2 S),
// entropy = ln2 * (log2 S - Q/S). M is not known while the row streams, so a
// thread sums against a reference that trails its running maximum and moves
// (one rescale of the sums) only when a logit passes it by 2^LAG: terms stay
// below 2^LAG, far inside fp32, and rescales are rare. Differences are taken
// before the multiply by k, so that rows at the type's lowest value (a fully
// masked row) do not overflow.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>
#include <math.h>

#include "common.cuh"
#include "token_loss.cuh"

namespace qs {
namespace loss {

constexpr int NT = 256;  // threads per CTA
constexpr int NW = NT / 32;
constexpr int U = 4;     // 16-byte loads in flight per thread
constexpr int MAXC = 8;  // CTAs of a row's cluster at most
constexpr float LAG = 20.0f;
constexpr float NEG = -FLT_MAX;
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

// ---- running sums of one thread -------------------------------------------

struct Acc {
    float ref;  // what the sums are taken against (NEG: nothing yet)
    float mx;   // largest element
    float s, q;
};

// Adds the N elements of x (their maximum is mx).
template <bool ENT, int N>
__device__ __forceinline__ void add(Acc& a, const float (&x)[N], float k) {
    float mx = x[0];
#pragma unroll
    for (int i = 1; i < N; i++) mx = fmaxf(mx, x[i]);
    if ((mx - a.ref) * k > LAG) {
        const float d = fmaxf((a.ref - mx) * k, -1e30f);  // finite, for sums still at 0
        const float f = ex2_approx(d);
        if (ENT) a.q = (a.q + a.s * d) * f;
        a.s *= f;
        a.ref = mx;
    }
    a.mx = fmaxf(a.mx, mx);
    const f32x2 nref = pack2(-a.ref, -a.ref), kk = pack2(k, k);
    f32x2 s = pack2(0.0f, 0.0f), q = pack2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        float t0, t1;
        unpack2(mul2(add2(pack2(x[i], x[i + 1]), nref), kk), t0, t1);
        const f32x2 e = pack2(ex2_approx(t0), ex2_approx(t1));
        s = add2(s, e);
        // a term of 0 at t = -inf must not become NaN; NaN stays in e
        if (ENT) q = fma2(e, pack2(fmaxf(t0, -200.0f), fmaxf(t1, -200.0f)), q);
    }
    float a0, a1;
    unpack2(s, a0, a1);
    a.s += a0 + a1;
    if (ENT) {
        unpack2(q, a0, a1);
        a.q += a0 + a1;
    }
}

// (max, sum, Q) of a set of elements, the sums taken against the maximum.
struct Part {
    double s, q;
    float m;
    float pad;
};

// Brings sums taken against `from` to `to` (>= from where the sums are not 0).
template <typename F>
__device__ __forceinline__ void rebase(F& s, F& q, float from, float to, float k) {
    const float base = to == -INFINITY ? 0.0f : to;
    const float d = fmaxf((from - base) * k, -1e30f);
    const float f = from == to ? 1.0f : ex2_approx(d);
    q = (q + s * (F)(from == to ? 0.0f : d)) * (F)f;
    s *= (F)f;
}

__device__ __forceinline__ Part warp_part(const Acc& a, float k) {
    Part p;
    p.m = warp_max(a.mx);
    float s = a.s, q = a.q;
    // an untouched thread (ref NEG, sums 0) and one of only -inf end at 0
    rebase(s, q, a.ref, p.m, k);
    p.s = warp_sum((double)s);
    p.q = warp_sum((double)q);
    return p;
}

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
__device__ __forceinline__ void remote_store(const void* local, uint32_t rank, const Part& p) {
    const uint32_t a = (uint32_t)__cvta_generic_to_shared(local);
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(r), "d"(p.s) : "memory");
    asm volatile("st.shared::cluster.f64 [%0+8], %1;" ::"r"(r), "d"(p.q) : "memory");
    asm volatile("st.shared::cluster.f32 [%0+16], %1;" ::"r"(r), "f"(p.m) : "memory");
}

// ---- the gradient of one slice ---------------------------------------------

// grad_v = 2^(d*k) * (a + b * d*k) + [v == target] * one
struct Coef {
    float m, a, b, one;
    int kind;  // 0 as above, 1 zeros, 2 NaN
};

// p_v = 2^t / S with t = d*k, ln p_v = ln2 * (t - log2 S), so
// (g_lp ([v==target] - p) - g_ent p (ln p + H)) / T has this form.
__device__ __forceinline__ Coef make_coef(double M, double S, double H, double g_lp, double g_ent, double inv_t) {
    Coef c;
    const double w = -inv_t / S;
    c.m = (float)M;
    c.a = (float)(w * (g_lp + (g_ent != 0.0 ? g_ent * (H - log(S)) : 0.0)));
    c.b = (float)(w * LN2 * g_ent);
    c.one = (float)(g_lp * inv_t);
    c.kind = S != S ? 2 : M == -INFINITY ? 1 : 0;
    return c;
}

template <bool ENT>
__device__ __forceinline__ float grad1(const Coef& c, float l, float k) {
    const float t = (l - c.m) * k;
    const float e = ex2_approx(t);
    return ENT ? e * fmaf(c.b, fmaxf(t, -200.0f), c.a) : e * c.a;
}

// Writes CTA `part` of `parts`' share of a row's gradient.
template <typename T, bool ENT>
__device__ __forceinline__ void grad_slice(const T* row, T* out, int V, int target, const Coef& c, float k, int part, int parts) {
    constexpr int N = Type<T>::N;
    const Span sp = span_of(row, V);
    const int tid = threadIdx.x;
    const float fill = c.kind == 2 ? NAN : 0.0f;
    if (part == 0 && tid < sp.head + sp.tail) {
        const int v = tid < sp.head ? tid : V - sp.tail + (tid - sp.head);
        put1(out + v, c.kind ? fill : grad1<ENT>(c, widen1(row[v]), k) + (v == target ? c.one : 0.0f));
    }
    const int lo = (int)((int64_t)sp.packs * part / parts), hi = (int)((int64_t)sp.packs * (part + 1) / parts);
    const uint4* src = reinterpret_cast<const uint4*>(row + sp.head);
    T* dst = out + sp.head;
    const bool same = ((uintptr_t)dst & 15) == 0;
    const int hot = target >= sp.head ? (target - sp.head) / N : -1;  // the target's pack (tail: none here)
    for (int v0 = lo + tid; v0 < hi; v0 += NT * U) {
        uint4 p[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (v0 + u * NT < hi && c.kind == 0) p[u] = load_pack(src + v0 + u * NT);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int v = v0 + u * NT;
            if (v >= hi) continue;
            float x[N];
            if (c.kind == 0) {
                widen(p[u], x, (T*)nullptr);
#pragma unroll
                for (int i = 0; i < N; i++) x[i] = grad1<ENT>(c, x[i], k);
                if (v == hot) {
                    const int j = (target - sp.head) % N;
#pragma unroll
                    for (int i = 0; i < N; i++)
                        if (i == j) x[i] += c.one;
                }
            } else {
#pragma unroll
                for (int i = 0; i < N; i++) x[i] = fill;
            }
            if (same)
                reinterpret_cast<uint4*>(dst)[v] = narrow(x, (T*)nullptr);
            else
#pragma unroll
                for (int i = 0; i < N; i++) put1(dst + (int64_t)v * N + i, x[i]);
        }
    }
}

// ---- kernels -----------------------------------------------------------------

// One cluster per row: log-probability, entropy, and with POLICY the policy
// loss and the gradient.
template <typename T, bool ENT, bool POLICY>
__global__ void __launch_bounds__(NT) rows_kernel(const Args a) {
    __shared__ Part parts[MAXC * NW];
    const int C = (int)cluster_size(), rank = (int)cluster_rank();
    const int r = (int)(blockIdx.x / C);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T* row = (const T*)a.logits + (int64_t)r * a.ld;
    const int target = a.targets[r];
    const float k = a.k;
    if (C > 1) cluster_arrive();  // the peers' shared memory is written below

    double weight = 1.0;
    if (POLICY) weight = a.weight ? (double)a.weight[r] : 1.0 / a.rows;
    const bool live = target >= 0 && weight != 0.0;
    const bool bad = target >= a.V;
    Coef c;
    c.m = c.a = c.b = c.one = 0.0f;
    c.kind = 1;
    float lt = 0.0f;
    Acc acc{NEG, -INFINITY, 0.0f, 0.0f};
    if (live && !bad) {
        constexpr int N = Type<T>::N;
        lt = widen1(row[target]);
        const Span sp = span_of(row, a.V);
        if (rank == 0 && tid < sp.head + sp.tail) {
            const float x[2] = {widen1(row[tid < sp.head ? tid : a.V - sp.tail + (tid - sp.head)]), -INFINITY};
            add<ENT>(acc, x, k);
        }
        const int lo = (int)((int64_t)sp.packs * rank / C), hi = (int)((int64_t)sp.packs * (rank + 1) / C);
        const uint4* src = reinterpret_cast<const uint4*>(row + sp.head);
        for (int v0 = lo + tid; v0 < hi; v0 += NT * U) {
            uint4 p[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                p[u] = make_uint4(Type<T>::NEG_INF, Type<T>::NEG_INF, Type<T>::NEG_INF, Type<T>::NEG_INF);
                if (v0 + u * NT < hi) p[u] = load_pack(src + v0 + u * NT);
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                float x[N];
                widen(p[u], x, (T*)nullptr);
                add<ENT>(acc, x, k);
            }
        }
    }
    const Part mine = warp_part(acc, k);
    if (C > 1) {
        cluster_wait();
        if (lane < C) remote_store(&parts[rank * NW + warp], lane, mine);
        cluster_arrive();
        cluster_wait();
    } else {
        if (lane == 0) parts[warp] = mine;
        __syncthreads();
    }
    // every warp joins the C * NW parts in the same order
    float M = -INFINITY;
    double S = 0.0, Q = 0.0;
    for (int i = lane; i < C * NW; i += 32) M = fmaxf(M, parts[i].m);
    M = warp_max(M);
    for (int i = lane; i < C * NW; i += 32) {
        Part p = parts[i];
        rebase(p.s, p.q, p.m, M, k);
        S += p.s, Q += p.q;
    }
    S = warp_sum(S), Q = warp_sum(Q);

    double lp = 0.0, H = 0.0, loss = 0.0;
    if (live) {
        const bool none = M == -INFINITY && S == 0.0;
        const double lnS = log(S);
        lp = none ? -INFINITY : (double)(lt - M) * ((double)k * LN2) - lnS;
        if (ENT) H = none ? 0.0 : lnS - LN2 * (Q / S);
        if (bad) lp = H = NAN;
        if (POLICY) {
            const double adv = a.adv[r], ratio = exp(lp - (double)a.old_lp[r]);
            const double lo = 1.0 - a.clip_lo, hi = 1.0 + a.clip_hi;
            const double fit = ratio < lo ? lo : ratio > hi ? hi : ratio;  // NaN stays
            const double x = ratio * adv, y = fit * adv;
            loss = x <= y ? -x : y < x ? -y : NAN;
            double g = x <= y ? -x : y < x ? 0.0 : NAN;
            if (a.kl != 0.0) {
                const double u = (double)a.ref_lp[r] - lp, eu = exp(u);
                loss += a.kl * (eu - u - 1.0);
                g += a.kl * (1.0 - eu);
            }
            if (ENT && a.ec != 0.0) loss -= a.ec * H;
            if (a.grad) {
                c = make_coef(M, S, H, g * weight * a.scale, ENT ? -a.ec * weight * a.scale : 0.0, a.inv_t);
                if (bad) c.kind = 2;
            }
        }
    }
    if (rank == 0 && tid == 0) {
        a.logprob[r] = (float)lp;
        if (a.entropy) a.entropy[r] = (float)H;
        if (a.stats) a.stats[r] = {live && !bad ? M : 0.0f, live && !bad ? (float)S : 0.0f};
        if (a.row_grad) a.row_grad[r] = 0.0f;
        if (POLICY) a.row_loss[r] = (float)loss;
    }
    if (POLICY && a.grad) grad_slice<T, ENT>(row, (T*)a.grad + (int64_t)r * a.grad_ld, a.V, target, c, k, rank, C);
}

// The gradient from given statistics and per-row derivatives; gridDim.y CTAs
// per row.
template <typename T, bool ENT>
__global__ void __launch_bounds__(NT) grad_kernel(const Args a) {
    const int r = (int)blockIdx.x;
    const int target = a.targets[r];
    Coef c;
    c.m = c.a = c.b = c.one = 0.0f;
    c.kind = 1;
    if (target >= a.V) {
        c.kind = 2;
    } else if (target >= 0) {
        const quasar_logprob_stat s = a.stats_in[r];
        c = make_coef(s.max, s.sum, ENT ? a.ent_in[r] : 0.0, a.g_lp[r], ENT ? a.g_ent[r] : 0.0, a.inv_t);
    }
    grad_slice<T, ENT>((const T*)a.logits + (int64_t)r * a.ld, (T*)a.grad + (int64_t)r * a.grad_ld, a.V, target, c, a.k,
                       (int)blockIdx.y, (int)gridDim.y);
}

// Sum over 128 threads, the same in every run; all threads get it.
__device__ __forceinline__ double cta_sum(double x, double* buf, int threads) {
    x = warp_sum(x);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = x;
    __syncthreads();
    double s = 0.0;
    for (int i = 0; i < threads / 32; i++) s += buf[i];
    return s;
}

// One CTA per pair.
__global__ void __launch_bounds__(128) pair_kernel(const PairArgs p) {
    __shared__ double buf[4];
    const int i = blockIdx.x, tid = threadIdx.x;
    const int at[3] = {p.cu[2 * i], p.cu[2 * i + 1], p.cu[2 * i + 2]};
    const bool ok = at[0] >= 0 && at[0] <= at[1] && at[1] <= at[2] && at[2] <= p.rows;
    double sum[2] = {0.0, 0.0}, n[2] = {0.0, 0.0};
    if (ok) {
        for (int s = 0; s < 2; s++) {
            double x = 0.0, c = 0.0;
            for (int r = at[s] + tid; r < at[s + 1]; r += 128)
                if (p.targets[r] >= 0) x += (double)p.logprob[r], c += 1.0;
            sum[s] = cta_sum(x, buf, 128);
            n[s] = cta_sum(c, buf, 128);
        }
    } else {
        sum[0] = sum[1] = NAN;
    }
    double score[2], by[2];
    for (int s = 0; s < 2; s++) {
        by[s] = p.mean && n[s] > 0.0 ? 1.0 / n[s] : 1.0;
        score[s] = sum[s] * by[s] - (p.ref ? (double)p.ref[2 * i + s] : 0.0);
    }
    const double x = p.beta * (score[0] - score[1]);
    // softplus(-x) and softplus(x); sigmoid(-x) and sigmoid(x)
    const double tail = log1p(exp(-fabs(x)));
    const double up = fmax(-x, 0.0) + tail, down = fmax(x, 0.0) + tail;
    const double sn = 1.0 / (1.0 + exp(x)), sp = 1.0 / (1.0 + exp(-x));
    const double loss = (1.0 - p.eps) * up + (p.eps != 0.0 ? p.eps * down : 0.0);
    const double w = p.weight ? (double)p.weight[i] : 1.0 / p.pairs;
    const double g = -p.beta * ((1.0 - p.eps) * sn - p.eps * sp) * w * p.scale;
    if (tid == 0) {
        p.seq[2 * i] = (float)sum[0];
        p.seq[2 * i + 1] = (float)sum[1];
        p.pair_loss[i] = (float)(x == x ? loss : NAN);
    }
    if (ok)
        for (int s = 0; s < 2; s++)
            for (int r = at[s] + tid; r < at[s + 1]; r += 128)
                if (p.targets[r] >= 0) p.row_grad[r] = (float)((s ? -g : g) * by[s]);
}

__global__ void __launch_bounds__(1024) weighted_sum_kernel(const float* x, const float* w, int n, float* out) {
    __shared__ double buf[32];
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 1024) {
        const double wi = w ? (double)w[i] : 1.0;
        if (wi != 0.0) s += wi * (double)x[i];
    }
    s = cta_sum(s, buf, 1024);
    if (threadIdx.x == 0) out[0] = (float)(w || n == 0 ? s : s / n);
}

// ---- launchers ---------------------------------------------------------------

// CTAs per row.
static int row_cluster(const Args& a) {
    int C = MAXC;
    while (C > 1 && (int64_t)a.rows * C > INT32_MAX) C /= 2;  // the grid's limit
    return C;
}

template <typename T, bool ENT, bool POLICY>
static cudaError_t rows_launch(const Args& a, cudaStream_t st) {
    const int C = row_cluster(a);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.rows * (unsigned)C);
    cfg.blockDim = dim3(NT);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = C;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, rows_kernel<T, ENT, POLICY>, a);
}

template <typename T>
static cudaError_t rows_typed(const Args& a, cudaStream_t st) {
    const bool ent = a.entropy != nullptr || a.ec != 0.0;
    if (a.adv) return ent ? rows_launch<T, true, true>(a, st) : rows_launch<T, false, true>(a, st);
    return ent ? rows_launch<T, true, false>(a, st) : rows_launch<T, false, false>(a, st);
}

cudaError_t launch_rows(const Args& a, int dtype, cudaStream_t st) {
    if (dtype == QUASAR_F32) return rows_typed<float>(a, st);
    if (dtype == QUASAR_F16) return rows_typed<__half>(a, st);
    return rows_typed<__nv_bfloat16>(a, st);
}

template <typename T>
static cudaError_t grad_typed(const Args& a, cudaStream_t st) {
    const dim3 grid((unsigned)a.rows, 8);
    if (a.g_ent)
        grad_kernel<T, true><<<grid, NT, 0, st>>>(a);
    else
        grad_kernel<T, false><<<grid, NT, 0, st>>>(a);
    return cudaPeekAtLastError();
}

cudaError_t launch_grad(const Args& a, int dtype, cudaStream_t st) {
    if (dtype == QUASAR_F32) return grad_typed<float>(a, st);
    if (dtype == QUASAR_F16) return grad_typed<__half>(a, st);
    return grad_typed<__nv_bfloat16>(a, st);
}

cudaError_t launch_pairs(const PairArgs& p, cudaStream_t st) {
    pair_kernel<<<p.pairs, 128, 0, st>>>(p);
    return cudaPeekAtLastError();
}

cudaError_t launch_weighted_sum(const float* x, const float* w, int n, float* out, cudaStream_t st) {
    weighted_sum_kernel<<<1, 1024, 0, st>>>(x, w, n, out);
    return cudaPeekAtLastError();
}

}  // namespace loss
}  // namespace qs
