// RMS norm of every query and key head followed by the position rotation, forward and backward, in one pass over the heads.
//
//   n  = x * rstd * g,  rstd = rsqrt(mean(x^2) + eps) over the head's D elements,  g = gamma (or 1 + gamma)
//   y  = n with its first R elements rotated by the angle of the token's position: for every pair (a, b),
//        y_a = n_a cos - n_b sin,  y_b = n_b cos + n_a sin.  Pairs are (i, i + R / 2), or (2 i, 2 i + 1) when interleaved;
//        the last D - R elements pass through.
//   backward:  dn = dy rotated back;  dgamma = sum over rows of dn * xhat (xhat = x * rstd);
//              dx = (dn * g - xhat * mean(dn * g * xhat)) * rstd.   rstd is recomputed from x, which is read anyway.
//
// Bound: HBM.  The forward reads and writes each head once, the backward reads x and dy and writes dx.  A head is owned by G
// neighbouring lanes and never leaves their registers: a lane holds whole pairs (the vectors at i and at i + R / 2), so the
// rotation needs no exchange and the norm one shuffle reduction.  A warp takes heads of one token only: the token's cosines and
// sines and the gains are converted once for all of them.  Arithmetic in fp32, one rounding at the end.
#include <algorithm>

#include "common.cuh"
#include "sm100_ptx.cuh"

namespace ptb {
using namespace sm100;

constexpr int kQkThreads = 128;
constexpr int kQkBwdThreads = 256;
constexpr int kQkMaxD = 1024;

struct QkArgs {
    const void *x[2], *dy[2], *gamma[2];   // [0] queries, [1] keys
    void *out[2];                          // forward: y; backward: dx.  Contiguous [T, heads, D]
    int64_t xb[2], xt[2], xh[2];           // strides of x in elements: batch, token, head
    int64_t gb[2], gt[2], gh[2];           // strides of dy (backward)
    int heads[2];
    int chunks[2];                         // warps per token: ceil(heads / heads per warp)
    const float *cos, *sin;                // [P, R / 2]
    const void *positions;                 // int32 / int64 [T], or null: the index inside the batch entry
    int pos_bytes;
    int64_t T, S, P;                       // tokens, tokens per batch entry, rows of the tables
    int D, R;
    float eps;
    float g0;                              // added to gamma: 1 when zero centred
    float *partial;                        // backward: [parts, D] sums of dn * xhat of every CTA (query CTAs first)
    int parts_q, parts;
    int *status;
};

template <typename T> __device__ __forceinline__ float qk_to_f(T v) { return (float) v; }
template <typename T> __device__ __forceinline__ T qk_from_f(float v);
template <> __device__ __forceinline__ float qk_from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 qk_from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half qk_from_f<__half>(float v) { return __float2half_rn(v); }

template <typename T, int V> struct alignas(sizeof(T) * V) QkVec { T e[V]; };

// Row of the tables of token t, or -1 (reported) when its position lies outside of them.
__device__ __forceinline__ int64_t qk_position(const QkArgs &a, int64_t t) {
    int64_t p = t % a.S;
    if (a.positions != nullptr)
        p = a.pos_bytes == 8 ? reinterpret_cast<const int64_t *>(a.positions)[t] : (int64_t) reinterpret_cast<const int *>(a.positions)[t];
    if (p < 0 || p >= a.P) {
        if (a.status != nullptr) *reinterpret_cast<volatile int *>(a.status) = PT_ERR_INVALID;
        return -1;
    }
    return p;
}

// What a lane owns of a head: ITEMS items of two vectors.  Neighbours half a rotation apart form an item in the half-split
// form (indices below NP), else the item just holds two vectors.
template <int V, int G, int ITEMS, bool IL> struct QkLane {
    int off[ITEMS][2];      // element offset of each vector; -1: none
    bool rot[ITEMS][2];     // the vector lies in the rotated part (half-split: both or none)
    __device__ __forceinline__ void init(int lane, int D, int R) {
        const int n_items = IL ? (D / V + 1) / 2 : R / 2 / V + ((D - R) / V + 1) / 2;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int idx = lane % G + i * G;
            int o0, o1;
            if constexpr (IL) {
                o0 = idx * V;
                o1 = (idx + n_items) * V;
            } else {
                const int np = R / 2 / V;
                o0 = idx < np ? idx * V : R + 2 * (idx - np) * V;
                o1 = idx < np ? R / 2 + idx * V : o0 + V;
            }
            off[i][0] = idx < n_items ? o0 : -1;
            off[i][1] = idx < n_items && o1 < D ? o1 : -1;
            rot[i][0] = off[i][0] >= 0 && o0 < R;
            rot[i][1] = off[i][1] >= 0 && o1 < R;
        }
    }
    // half-split: cs[i][e] belongs to pair e of the item; interleaved: cs[i][0 .. V/2) to the first vector, the rest to the second
    __device__ __forceinline__ void load_table(const float *row, float (&c)[ITEMS][V]) const {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            if constexpr (IL) {
#pragma unroll
                for (int v = 0; v < 2; ++v)
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) c[i][v * (V / 2) + e] = rot[i][v] ? row[off[i][v] / 2 + e] : 0.f;
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) c[i][e] = rot[i][0] ? row[off[i][0] + e] : 0.f;
            }
        }
    }
    // rotation of the item's two vectors (sign = -1: back)
    __device__ __forceinline__ void rotate(int i, float (&a)[V], float (&b)[V], const float (&c)[ITEMS][V], const float (&s)[ITEMS][V], float sign) const {
        if constexpr (IL) {
#pragma unroll
            for (int e = 0; e < V; e += 2) {
                const float ca = c[i][e / 2], sa = sign * s[i][e / 2], cb = c[i][V / 2 + e / 2], sb = sign * s[i][V / 2 + e / 2];
                const float a0 = a[e] * ca - a[e + 1] * sa, a1 = a[e + 1] * ca + a[e] * sa;
                const float b0 = b[e] * cb - b[e + 1] * sb, b1 = b[e + 1] * cb + b[e] * sb;
                if (rot[i][0]) { a[e] = a0; a[e + 1] = a1; }
                if (rot[i][1]) { b[e] = b0; b[e + 1] = b1; }
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float ce = c[i][e], se = sign * s[i][e];
                const float a0 = a[e] * ce - b[e] * se, b0 = b[e] * ce + a[e] * se;
                if (rot[i][0]) { a[e] = a0; b[e] = b0; }
            }
        }
    }
};

template <int G> __device__ __forceinline__ float qk_group_sum(float v) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// A warp takes 32 / G * U heads of one token, U per lane group, their loads all in flight together.
template <typename T, int V, int G, int ITEMS, bool IL, int U>
__global__ void __launch_bounds__(kQkThreads) qk_norm_rope_fwd_kernel(QkArgs a) {
    constexpr int kRows = 32 / G;
    using Vt = QkVec<T, V>;
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31;
    const int per_token = a.chunks[0] + a.chunks[1];
    const int64_t unit = (int64_t) blockIdx.x * (kQkThreads / 32) + (threadIdx.x >> 5);
    const int64_t t = unit / per_token;
    if (t >= a.T) return;
    int chunk = (int) (unit - t * per_token);
    const int r = chunk >= a.chunks[0];
    chunk -= r ? a.chunks[0] : 0;
    const int h0 = chunk * kRows * U + lane / G;
    const int64_t b = t / a.S, ti = t - b * a.S;
    const T *x = reinterpret_cast<const T *>(a.x[r]) + b * a.xb[r] + ti * a.xt[r];
    QkLane<V, G, ITEMS, IL> ln;
    ln.init(lane, a.D, a.R);

    Vt raw[U][ITEMS][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int h = h0 + u * kRows;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                raw[u][i][v] = Vt{};
                if (h < a.heads[r] && ln.off[i][v] >= 0) raw[u][i][v] = *reinterpret_cast<const Vt *>(x + (int64_t) h * a.xh[r] + ln.off[i][v]);
            }
    }
    const int64_t pos = qk_position(a, t);
    float c[ITEMS][V], s[ITEMS][V], g[ITEMS][2][V];
    ln.load_table(a.cos + (pos < 0 ? 0 : pos) * (a.R / 2), c);
    ln.load_table(a.sin + (pos < 0 ? 0 : pos) * (a.R / 2), s);
    const T *gamma = reinterpret_cast<const T *>(a.gamma[r]);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            Vt gr = {};
            if (ln.off[i][v] >= 0) gr = *reinterpret_cast<const Vt *>(gamma + ln.off[i][v]);
#pragma unroll
            for (int e = 0; e < V; ++e) g[i][v][e] = qk_to_f<T>(gr.e[e]) + a.g0;
        }

    T *out = reinterpret_cast<T *>(a.out[r]) + t * a.heads[r] * a.D;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int v = 0; v < 2; ++v)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float f = qk_to_f<T>(raw[u][i][v].e[e]);
                    ss += f * f;
                }
        const float rstd = rsqrtf(qk_group_sum<G>(ss) / (float) a.D + a.eps);
        const int h = h0 + u * kRows;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            float n[2][V];
#pragma unroll
            for (int v = 0; v < 2; ++v)
#pragma unroll
                for (int e = 0; e < V; ++e) n[v][e] = qk_to_f<T>(raw[u][i][v].e[e]) * rstd * g[i][v][e];
            ln.rotate(i, n[0], n[1], c, s, 1.f);
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                if (h >= a.heads[r] || ln.off[i][v] < 0) continue;
                Vt o;
#pragma unroll
                for (int e = 0; e < V; ++e) o.e[e] = qk_from_f<T>(pos < 0 ? 0.f : n[v][e]);
                *reinterpret_cast<Vt *>(out + (int64_t) h * a.D + ln.off[i][v]) = o;
            }
        }
    }
}

// Persistent CTAs: the first parts_q work on queries, the rest on keys, so that a lane's share of dgamma stays in registers over
// all its heads.  Per CTA one row of partial sums (fixed order: lanes, then warps); qk_dgamma_kernel adds the rows.
template <typename T, int V, int G, int ITEMS, bool IL, int U>
__global__ void __launch_bounds__(kQkBwdThreads) qk_norm_rope_bwd_kernel(QkArgs a) {
    constexpr int kRows = 32 / G;
    constexpr int kWarps = kQkBwdThreads / 32;
    using Vt = QkVec<T, V>;
    extern __shared__ float s_part[];   // [warps][D]
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r = (int) blockIdx.x >= a.parts_q;
    const int cta = (int) blockIdx.x - (r ? a.parts_q : 0), ctas = r ? a.parts - a.parts_q : a.parts_q;
    const int64_t units = a.T * a.chunks[r];
    QkLane<V, G, ITEMS, IL> ln;
    ln.init(lane, a.D, a.R);
    float g[ITEMS][2][V], dg[ITEMS][2][V];
    const T *gamma = reinterpret_cast<const T *>(a.gamma[r]);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            Vt gr = {};
            if (ln.off[i][v] >= 0) gr = *reinterpret_cast<const Vt *>(gamma + ln.off[i][v]);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                g[i][v][e] = qk_to_f<T>(gr.e[e]) + a.g0;
                dg[i][v][e] = 0.f;
            }
        }
    for (int64_t unit = (int64_t) cta * kWarps + warp; unit < units; unit += (int64_t) ctas * kWarps) {
        const int64_t t = unit / a.chunks[r];
        const int h0 = (int) (unit - t * a.chunks[r]) * kRows * U + lane / G;
        const int64_t b = t / a.S, ti = t - b * a.S;
        const T *x = reinterpret_cast<const T *>(a.x[r]) + b * a.xb[r] + ti * a.xt[r];
        const T *dy = reinterpret_cast<const T *>(a.dy[r]) + b * a.gb[r] + ti * a.gt[r];
        Vt rx[U][ITEMS][2], rd[U][ITEMS][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = h0 + u * kRows;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    rx[u][i][v] = Vt{};
                    rd[u][i][v] = Vt{};
                    if (h < a.heads[r] && ln.off[i][v] >= 0) {
                        rx[u][i][v] = *reinterpret_cast<const Vt *>(x + (int64_t) h * a.xh[r] + ln.off[i][v]);
                        rd[u][i][v] = *reinterpret_cast<const Vt *>(dy + (int64_t) h * a.gh[r] + ln.off[i][v]);
                    }
                }
        }
        const int64_t pos = qk_position(a, t);
        float c[ITEMS][V], s[ITEMS][V];
        ln.load_table(a.cos + (pos < 0 ? 0 : pos) * (a.R / 2), c);
        ln.load_table(a.sin + (pos < 0 ? 0 : pos) * (a.R / 2), s);
        T *dx = reinterpret_cast<T *>(a.out[r]) + t * a.heads[r] * a.D;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = h0 + u * kRows;
            float ss = 0.f, dot = 0.f;
            float dn[ITEMS][2][V];
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
                for (int v = 0; v < 2; ++v)
#pragma unroll
                    for (int e = 0; e < V; ++e) dn[i][v][e] = qk_to_f<T>(rd[u][i][v].e[e]);
                ln.rotate(i, dn[i][0], dn[i][1], c, s, -1.f);
#pragma unroll
                for (int v = 0; v < 2; ++v)
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float f = qk_to_f<T>(rx[u][i][v].e[e]);
                        ss += f * f;
                        dot += dn[i][v][e] * g[i][v][e] * f;
                    }
            }
            const float rstd = rsqrtf(qk_group_sum<G>(ss) / (float) a.D + a.eps);
            const float m = qk_group_sum<G>(dot) * rstd / (float) a.D;   // mean(dn * g * xhat)
            if (h >= a.heads[r]) continue;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    if (ln.off[i][v] < 0) continue;
                    Vt o;
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float xh = qk_to_f<T>(rx[u][i][v].e[e]) * rstd;
                        o.e[e] = qk_from_f<T>(pos < 0 ? 0.f : (dn[i][v][e] * g[i][v][e] - xh * m) * rstd);
                        if (pos >= 0) dg[i][v][e] += dn[i][v][e] * xh;
                    }
                    *reinterpret_cast<Vt *>(dx + (int64_t) h * a.D + ln.off[i][v]) = o;
                }
        }
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float d = dg[i][v][e];
#pragma unroll
                for (int o = G; o < 32; o <<= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
                if (lane < G && ln.off[i][v] >= 0) s_part[warp * a.D + ln.off[i][v] + e] = d;
            }
    __syncthreads();
    for (int d = threadIdx.x; d < a.D; d += kQkBwdThreads) {
        float acc = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) acc += s_part[w * a.D + d];
        a.partial[(int64_t) blockIdx.x * a.D + d] = acc;
    }
}

// Any D, R and alignment: a warp per head, element-wise accesses, each lane owning whole pairs (and elements of the rest).
// Serves the layouts the vector kernels do not (rows or halves that are not a multiple of two elements or not aligned).
template <typename T, bool BWD>
__global__ void __launch_bounds__(kQkBwdThreads) qk_norm_rope_any_kernel(QkArgs a, int interleaved) {
    constexpr int kWarps = kQkBwdThreads / 32;
    extern __shared__ float s_part[];   // BWD: [warps][D] sums of dn * xhat
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int half = a.R / 2, n_items = half + (a.D - a.R);
    float *mine = s_part + warp * a.D;
    if constexpr (BWD) {
        for (int d = lane; d < a.D; d += 32) mine[d] = 0.f;
        __syncwarp();
    }
    // forward: units are heads of queries and keys together; backward: of the CTA's side alone
    const int r_cta = BWD ? (int) blockIdx.x >= a.parts_q : 0;
    const int cta = BWD && r_cta ? (int) blockIdx.x - a.parts_q : (int) blockIdx.x;
    const int ctas = BWD ? (r_cta ? a.parts - a.parts_q : a.parts_q) : (int) gridDim.x;
    const int per_token = BWD ? a.heads[r_cta] : a.heads[0] + a.heads[1];
    for (int64_t unit = (int64_t) cta * kWarps + warp; unit < a.T * per_token; unit += (int64_t) ctas * kWarps) {
        const int64_t t = unit / per_token;
        int h = (int) (unit - t * per_token);
        const int r = BWD ? r_cta : h >= a.heads[0];
        if (!BWD && r) h -= a.heads[0];
        const int64_t b = t / a.S, ti = t - b * a.S, pos = qk_position(a, t);
        const T *x = reinterpret_cast<const T *>(a.x[r]) + b * a.xb[r] + ti * a.xt[r] + (int64_t) h * a.xh[r];
        const T *dy = BWD ? reinterpret_cast<const T *>(a.dy[r]) + b * a.gb[r] + ti * a.gt[r] + (int64_t) h * a.gh[r] : nullptr;
        const T *gamma = reinterpret_cast<const T *>(a.gamma[r]);
        T *out = reinterpret_cast<T *>(a.out[r]) + (t * a.heads[r] + h) * a.D;
        const float *cr = a.cos + (pos < 0 ? 0 : pos) * half, *sr = a.sin + (pos < 0 ? 0 : pos) * half;
        auto at = [&](int i, int &p, int &q) {   // elements of item i: a pair, or one element (q < 0)
            if (i < half) { p = interleaved ? 2 * i : i; q = interleaved ? 2 * i + 1 : i + half; }
            else { p = a.R + (i - half); q = -1; }
        };
        auto turned_back = [&](int i, int p, int q, float &dp, float &dq) {
            dp = qk_to_f<T>(dy[p]);
            dq = q < 0 ? 0.f : qk_to_f<T>(dy[q]);
            if (q >= 0) {
                const float u = dp * cr[i] + dq * sr[i], w = dq * cr[i] - dp * sr[i];
                dp = u; dq = w;
            }
        };
        float ss = 0.f, dot = 0.f;
        for (int i = lane; i < n_items; i += 32) {
            int p, q;
            at(i, p, q);
            const float fp = qk_to_f<T>(x[p]), fq = q < 0 ? 0.f : qk_to_f<T>(x[q]);
            ss += fp * fp + fq * fq;
            if constexpr (BWD) {
                float dp, dq;
                turned_back(i, p, q, dp, dq);
                dot += dp * (qk_to_f<T>(gamma[p]) + a.g0) * fp;
                if (q >= 0) dot += dq * (qk_to_f<T>(gamma[q]) + a.g0) * fq;
            }
        }
        const float rstd = rsqrtf(qk_group_sum<32>(ss) / (float) a.D + a.eps);
        const float m = BWD ? qk_group_sum<32>(dot) * rstd / (float) a.D : 0.f;
        for (int i = lane; i < n_items; i += 32) {
            int p, q;
            at(i, p, q);
            const float gp = qk_to_f<T>(gamma[p]) + a.g0, gq = q < 0 ? 0.f : qk_to_f<T>(gamma[q]) + a.g0;
            const float xp = qk_to_f<T>(x[p]) * rstd, xq = q < 0 ? 0.f : qk_to_f<T>(x[q]) * rstd;
            float op, oq = 0.f;
            if constexpr (BWD) {
                float dp, dq;
                turned_back(i, p, q, dp, dq);
                op = (dp * gp - xp * m) * rstd;
                oq = (dq * gq - xq * m) * rstd;
                if (pos >= 0) {
                    mine[p] += dp * xp;
                    if (q >= 0) mine[q] += dq * xq;
                }
            } else {
                op = xp * gp;
                if (q >= 0) {
                    const float np = op, nq = xq * gq;
                    op = np * cr[i] - nq * sr[i];
                    oq = nq * cr[i] + np * sr[i];
                }
            }
            out[p] = qk_from_f<T>(pos < 0 ? 0.f : op);
            if (q >= 0) out[q] = qk_from_f<T>(pos < 0 ? 0.f : oq);
        }
    }
    if constexpr (BWD) {
        __syncthreads();
        for (int d = threadIdx.x; d < a.D; d += kQkBwdThreads) {
            float acc = 0.f;
            for (int w = 0; w < kWarps; ++w) acc += s_part[w * a.D + d];
            a.partial[(int64_t) blockIdx.x * a.D + d] = acc;
        }
    }
}

// dgamma = sum of the partial rows of its side, in a fixed order; blockIdx.y: 0 queries, 1 keys.
template <typename T>
__global__ void __launch_bounds__(512) qk_dgamma_kernel(const float *__restrict__ partial, int parts_q, int parts, int D, T *dq_gamma, T *dk_gamma) {
    __shared__ float s_sum[16][33];
    grid_dep_wait();
    const int c = threadIdx.x & 31, lane = threadIdx.x >> 5, d = (int) blockIdx.x * 32 + c;
    const int first = blockIdx.y ? parts_q : 0, last = blockIdx.y ? parts : parts_q;
    float acc = 0.f;
    if (d < D)
#pragma unroll 4
        for (int p = first + lane; p < last; p += 16) acc += partial[(int64_t) p * D + d];
    s_sum[lane][c] = acc;
    __syncthreads();
    if (lane == 0 && d < D) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) t += s_sum[i][c];
        (blockIdx.y ? dk_gamma : dq_gamma)[d] = qk_from_f<T>(t);
    }
}

// ------------------------------------------------------------------------------------------------ host side
// How a head is laid over lanes.  vec elements per access: a full 16 bytes when the head, both halves of the rotation and every
// stride are whole vectors; else two elements; 0: the element-wise kernel.
static int qk_vec(const QkArgs &a, int esize, bool il, bool bwd) {
    for (int v : {16 / esize, 2}) {
        bool ok = a.D % v == 0 && (il ? a.R : a.R / 2) % v == 0 && a.R % v == 0;
        for (int r = 0; r < 2; ++r) {
            ok = ok && aligned(a.x[r], v * esize) && aligned(a.gamma[r], v * esize) && aligned(a.out[r], v * esize) &&
                 (a.xb[r] | a.xt[r] | a.xh[r]) % v == 0;
            if (bwd) ok = ok && aligned(a.dy[r], v * esize) && (a.gb[r] | a.gt[r] | a.gh[r]) % v == 0;
        }
        const int items = il ? (a.D / v + 1) / 2 : a.R / 2 / v + ((a.D - a.R) / v + 1) / 2;
        if (ok && items <= (v == 2 ? 64 : 32)) return v;
    }
    return 0;
}

template <typename T, int V, int G, int ITEMS, bool IL> static int qk_launch(QkArgs a, bool bwd, cudaStream_t st) {
    // heads per lane group and warp: four while a token has that many (their loads overlap), one otherwise
    constexpr int kRows = 32 / G;
    if (!bwd) {
        const int most = std::max(a.heads[0], a.heads[1]);
        const int U = most >= 2 * kRows && ITEMS == 1 ? 4 : 1;
        for (int r = 0; r < 2; ++r) a.chunks[r] = (int) ceil_div(a.heads[r], kRows * U);
        const int64_t grid = ceil_div(a.T * (a.chunks[0] + a.chunks[1]), kQkThreads / 32);
        PT_REQUIRE(grid < (1ll << 31), "qk_norm_rope: too many tokens");
        if (U == 4) PT_CUDA_OK(launch_overlapped(qk_norm_rope_fwd_kernel<T, V, G, ITEMS, IL, ITEMS == 1 ? 4 : 1>, dim3((unsigned) grid), dim3(kQkThreads), 0, st, a));
        else PT_CUDA_OK(launch_overlapped(qk_norm_rope_fwd_kernel<T, V, G, ITEMS, IL, 1>, dim3((unsigned) grid), dim3(kQkThreads), 0, st, a));
        return PT_OK;
    }
    constexpr int U = ITEMS == 1 ? 2 : 1;
    for (int r = 0; r < 2; ++r) a.chunks[r] = (int) ceil_div(a.heads[r], kRows * U);
    PT_CUDA_OK(launch_overlapped(qk_norm_rope_bwd_kernel<T, V, G, ITEMS, IL, U>, dim3(a.parts), dim3(kQkBwdThreads),
                                 (size_t) (kQkBwdThreads / 32) * a.D * 4, st, a));
    return PT_OK;
}

template <typename T, bool IL> static int qk_dispatch(const QkArgs &a, bool bwd, cudaStream_t st) {
    constexpr int V16 = 16 / (int) sizeof(T);
    const int v = qk_vec(a, sizeof(T), IL, bwd);
    if (v == 0) {
        const size_t smem = bwd ? (size_t) (kQkBwdThreads / 32) * a.D * 4 : 0;
        const int64_t fwd_grid = std::min<int64_t>(ceil_div(a.T * (a.heads[0] + a.heads[1]), kQkBwdThreads / 32), (int64_t) sm_count() * 8);
        if (bwd) PT_CUDA_OK(launch_overlapped(qk_norm_rope_any_kernel<T, true>, dim3(a.parts), dim3(kQkBwdThreads), smem, st, a, (int) IL));
        else PT_CUDA_OK(launch_overlapped(qk_norm_rope_any_kernel<T, false>, dim3((unsigned) fwd_grid), dim3(kQkBwdThreads), smem, st, a, (int) IL));
        return PT_OK;
    }
    const int items = IL ? (a.D / v + 1) / 2 : a.R / 2 / v + ((a.D - a.R) / v + 1) / 2;
    if (v == V16) {
        if (items <= 4) return qk_launch<T, V16, 4, 1, IL>(a, bwd, st);
        if (items <= 8) return qk_launch<T, V16, 8, 1, IL>(a, bwd, st);
        if (items <= 16) return qk_launch<T, V16, 16, 1, IL>(a, bwd, st);
        return qk_launch<T, V16, 32, 1, IL>(a, bwd, st);
    }
    if (items <= 16) return qk_launch<T, 2, 16, 1, IL>(a, bwd, st);
    if (items <= 32) return qk_launch<T, 2, 32, 1, IL>(a, bwd, st);
    return qk_launch<T, 2, 32, 2, IL>(a, bwd, st);
}

static int qk_check(const QkArgs &a, int dtype, int64_t B) {
    PT_REQUIRE(dtype == PT_BF16 || dtype == PT_F16 || dtype == PT_F32, "qk_norm_rope: unsupported dtype %d", dtype);
    PT_REQUIRE(B >= 0 && a.S >= 0 && a.heads[0] >= 0 && a.heads[1] >= 0, "qk_norm_rope: negative extent");
    PT_REQUIRE(a.D >= 1 && a.D <= kQkMaxD && a.R >= 0 && a.R % 2 == 0 && a.R <= a.D,
               "qk_norm_rope: the head size must lie in [1, %d] and the rotated part be even and no larger (got %d, %d)", kQkMaxD, a.D, a.R);
    PT_REQUIRE(a.pos_bytes == 0 || a.pos_bytes == 4 || a.pos_bytes == 8, "qk_norm_rope: positions must be int32 or int64");
    PT_REQUIRE((a.pos_bytes == 0) == (a.positions == nullptr), "qk_norm_rope: positions and their size go together");
    for (int r = 0; r < 2; ++r)
        PT_REQUIRE(a.T == 0 || a.heads[r] == 0 || (a.x[r] && a.out[r] && a.gamma[r]), "qk_norm_rope: null pointer");
    PT_REQUIRE(a.T == 0 || a.R == 0 || (a.cos && a.sin), "qk_norm_rope: null table");
    return PT_OK;
}

static int qk_parts(int64_t T, int Hq, int Hk, int &parts_q) {
    // CTAs of the backward: three per SM, shared between queries and keys by their heads, one at least for each side
    const int total = (int) std::max<int64_t>(2, std::min<int64_t>((int64_t) sm_count() * 3, ceil_div(T * (Hq + Hk), 16)));
    parts_q = Hq + Hk == 0 ? 1 : (int) std::min<int64_t>(total - 1, std::max<int64_t>(1, (int64_t) total * Hq / (Hq + Hk)));
    return total;
}

}  // namespace ptb

using namespace ptb;

extern "C" {

int pt_qk_norm_rope_fwd(const void *q, const void *k, int dtype, const void *q_gamma, const void *k_gamma, const float *cos, const float *sin,
                        const void *positions, int pos_bytes, int64_t B, int64_t S, int64_t P, int Hq, int Hk, int D, int R,
                        const int64_t *q_strides, const int64_t *k_strides, float eps, int interleaved, int zero_centered, void *q_out,
                        void *k_out, int *status, void *stream) {
    QkArgs a{};
    PT_REQUIRE(q_strides && k_strides, "qk_norm_rope: strides required");
    a.x[0] = q; a.x[1] = k; a.gamma[0] = q_gamma; a.gamma[1] = k_gamma; a.out[0] = q_out; a.out[1] = k_out;
    a.xb[0] = q_strides[0]; a.xt[0] = q_strides[1]; a.xh[0] = q_strides[2];
    a.xb[1] = k_strides[0]; a.xt[1] = k_strides[1]; a.xh[1] = k_strides[2];
    a.heads[0] = Hq; a.heads[1] = Hk; a.cos = cos; a.sin = sin; a.positions = positions; a.pos_bytes = pos_bytes;
    a.T = B * S; a.S = S; a.P = P; a.D = D; a.R = R; a.eps = eps; a.g0 = zero_centered ? 1.f : 0.f; a.status = status;
    const int rc = qk_check(a, dtype, B);
    if (rc != PT_OK) return rc;
    if (a.T == 0 || Hq + Hk == 0) return PT_OK;
    PT_SWITCH_SRC(dtype, T, return interleaved ? qk_dispatch<T, true>(a, false, (cudaStream_t) stream) : qk_dispatch<T, false>(a, false, (cudaStream_t) stream));
    return PT_OK;
}

int pt_qk_norm_rope_bwd_parts(int64_t T, int Hq, int Hk) {
    int parts_q;
    return qk_parts(T, Hq, Hk, parts_q);
}

int pt_qk_norm_rope_bwd(const void *dq, const void *dk, const void *q, const void *k, int dtype, const void *q_gamma, const void *k_gamma,
                        const float *cos, const float *sin, const void *positions, int pos_bytes, int64_t B, int64_t S, int64_t P, int Hq,
                        int Hk, int D, int R, const int64_t *dq_strides, const int64_t *dk_strides, const int64_t *q_strides,
                        const int64_t *k_strides, float eps, int interleaved, int zero_centered, void *dq_in, void *dk_in, void *dq_gamma,
                        void *dk_gamma, float *partial, int parts, int *status, void *stream) {
    QkArgs a{};
    PT_REQUIRE(q_strides && k_strides && dq_strides && dk_strides, "qk_norm_rope backward: strides required");
    a.x[0] = q; a.x[1] = k; a.dy[0] = dq; a.dy[1] = dk; a.gamma[0] = q_gamma; a.gamma[1] = k_gamma; a.out[0] = dq_in; a.out[1] = dk_in;
    a.xb[0] = q_strides[0]; a.xt[0] = q_strides[1]; a.xh[0] = q_strides[2];
    a.xb[1] = k_strides[0]; a.xt[1] = k_strides[1]; a.xh[1] = k_strides[2];
    a.gb[0] = dq_strides[0]; a.gt[0] = dq_strides[1]; a.gh[0] = dq_strides[2];
    a.gb[1] = dk_strides[0]; a.gt[1] = dk_strides[1]; a.gh[1] = dk_strides[2];
    a.heads[0] = Hq; a.heads[1] = Hk; a.cos = cos; a.sin = sin; a.positions = positions; a.pos_bytes = pos_bytes;
    a.T = B * S; a.S = std::max<int64_t>(S, 1); a.P = P; a.D = D; a.R = R; a.eps = eps; a.g0 = zero_centered ? 1.f : 0.f; a.status = status;
    const int rc = qk_check(a, dtype, B);
    if (rc != PT_OK) return rc;
    for (int r = 0; r < 2; ++r) PT_REQUIRE(a.T == 0 || a.heads[r] == 0 || a.dy[r], "qk_norm_rope backward: null pointer");
    a.parts = qk_parts(a.T, Hq, Hk, a.parts_q);
    PT_REQUIRE(partial && dq_gamma && dk_gamma && parts == a.parts, "qk_norm_rope backward: dgamma buffers / part count");
    a.partial = partial;
    cudaStream_t st = (cudaStream_t) stream;
    // with no tokens the CTAs still write their rows of zeros, and dgamma comes out as zero
    PT_SWITCH_SRC(dtype, T, {
        const int rc2 = interleaved ? qk_dispatch<T, true>(a, true, st) : qk_dispatch<T, false>(a, true, st);
        if (rc2 != PT_OK) return rc2;
        PT_CUDA_OK(launch_overlapped(qk_dgamma_kernel<T>, dim3((unsigned) ceil_div(D, 32), 2), dim3(512), 0, st, (const float *) partial, a.parts_q, a.parts, D,
                                     (T *) dq_gamma, (T *) dk_gamma));
    });
    return PT_OK;
}

}  // extern "C"
