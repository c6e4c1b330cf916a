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
// Measured (B200): forward 8192 x 72 heads of 128, bf16, 59.7 us (5.1 TB/s); forward and backward of 8191 x 40 heads, fp16, half
// rotated, 94.1 us (4.5 TB/s of the five passes); fp32, 8192 x 40 heads 52.3 us (6.4 TB/s) and 135 (6.2).  Issue slots are 0.69 and
// 0.62 busy and loads in flight bound the rest.  Heads that take two elements an access for four (R / 2 not a multiple of four)
// cost 1.5 times the time.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "gemm_common.cuh"
#include "sm100_ptx.cuh"

namespace ptb {
using namespace sm100;

constexpr int kQkThreads = 128;
constexpr int kQkBwdThreads = 256;
// CTAs per SM the registers are cut to.  Measured on 8192 x 72 heads of 128, bf16 (forward) and 8191 x 40 heads, fp16 (forward and
// backward): 8 and 3 CTAs 64.5 / 104.7 us; 6 and 3 69.3 / 125; 10 and 4 66.1 / 138; 8 and 2 65.4 / 142.  A few spilled registers
// cost less than the loads in flight that they buy.
constexpr int kQkFwdCtas = 8, kQkBwdCtas = 3;
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
    float eps, inv_d;                      // 1 / D
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

// ---------------------------------------------------------------- two fp32 values in one instruction
// The kernels are bound by instruction issue before they are bound by memory (29 instructions per element in scalar form), so
// the arithmetic runs on register pairs.
struct F2 { uint64_t v; };
__device__ __forceinline__ F2 f2(float x, float y) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void f2_split(F2 a, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a.v)); }
__device__ __forceinline__ F2 f2_swap(F2 a) {
    float x, y;
    f2_split(a, x, y);
    return f2(y, x);
}
__device__ __forceinline__ F2 f2_mul(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ float f2_sum(F2 a) {
    float x, y;
    f2_split(a, x, y);
    return x + y;
}

// V (2 or 4) elements of a head as they lie in memory, and as V / 2 pairs.  Heads are read and written once, with streaming accesses: the tables
// keep their place in the caches (8192 x 72 heads 62.6 -> 59.7 us, 8191 x 40 forward + backward 99.3 -> 94.1).
template <typename T, int V> struct QkWords { uint32_t w[V * sizeof(T) / 4]; };
template <typename T, int V> __device__ __forceinline__ QkWords<T, V> qk_load(const T *p) {
    QkWords<T, V> r;
    if constexpr (sizeof(r) == 4) r.w[0] = __ldcs(reinterpret_cast<const uint32_t *>(p));
    else if constexpr (sizeof(r) == 8) { const uint2 u = __ldcs(reinterpret_cast<const uint2 *>(p)); r.w[0] = u.x; r.w[1] = u.y; }
    else { const uint4 u = __ldcs(reinterpret_cast<const uint4 *>(p)); r.w[0] = u.x; r.w[1] = u.y; r.w[2] = u.z; r.w[3] = u.w; }
    return r;
}
template <typename T, int V> __device__ __forceinline__ F2 qk_pair(const QkWords<T, V> &r, int j) {
    if constexpr (sizeof(T) == 4) return f2(__uint_as_float(r.w[2 * j]), __uint_as_float(r.w[2 * j + 1]));
    else return f2(lo_f32<T>(r.w[j]), hi_f32<T>(r.w[j]));
}
template <typename T> __device__ __forceinline__ uint32_t qk_pack(F2 a) {
    float x, y;
    f2_split(a, x, y);
    return pack2<T>(x, y);
}
template <typename T, int V> __device__ __forceinline__ void qk_store(T *p, const F2 (&y)[V / 2]) {
    if constexpr (sizeof(T) == 4) {
        if constexpr (V == 2) {
            __stcs(reinterpret_cast<unsigned long long *>(p), (unsigned long long) y[0].v);
        } else {
            float4 w;
            f2_split(y[0], w.x, w.y);
            f2_split(y[1], w.z, w.w);
            __stcs(reinterpret_cast<float4 *>(p), w);
        }
    } else {
        if constexpr (V == 2) __stcs(reinterpret_cast<uint32_t *>(p), qk_pack<T>(y[0]));
        else __stcs(reinterpret_cast<uint2 *>(p), make_uint2(qk_pack<T>(y[0]), qk_pack<T>(y[1])));
    }
}

// Row of the tables of token t (ti: its index inside its batch entry), or -1 (reported) when its position lies outside of them.
__device__ __forceinline__ int64_t qk_position(const QkArgs &a, uint32_t t, uint32_t ti) {
    int64_t p = ti;
    if (a.pos_bytes == 8) p = reinterpret_cast<const int64_t *>(a.positions)[t];
    else if (a.pos_bytes == 4) p = reinterpret_cast<const int *>(a.positions)[t];
    if (p < 0 || p >= a.P) {
        report_status(a.status, PT_ERR_INVALID);
        return -1;
    }
    return p;
}

// What a lane owns of a head: ITEMS items of two vectors of V elements.  Half-split form: the vectors at i and at i + R / 2 form
// an item, so that both elements of every pair are the lane's own; what is not rotated is paired up anyhow.  Interleaved form: the
// pairs lie inside a vector.
template <typename T, int V, int G, int ITEMS, bool IL> struct QkLane {
    static constexpr int P = V / 2;   // register pairs of a vector
    int off[ITEMS][2];                // element offset of each vector; -1: none
    bool rot[ITEMS][2];               // the vector lies in the rotated part (half-split: both or none)
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
    // cosines and signed sines of every register pair: the pair becomes x * c + partner(x) * s (turned by -sign)
    __device__ __forceinline__ void load_table(const float *cos_row, const float *sin_row, float sign, F2 (&c)[ITEMS][2][P], F2 (&s)[ITEMS][2][P]) const {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            if constexpr (IL) {
#pragma unroll
                for (int v = 0; v < 2; ++v)
#pragma unroll
                    for (int j = 0; j < P; ++j) {
                        const float ce = rot[i][v] ? cos_row[off[i][v] / 2 + j] : 1.f, se = rot[i][v] ? sign * sin_row[off[i][v] / 2 + j] : 0.f;
                        c[i][v][j] = f2(ce, ce);
                        s[i][v][j] = f2(-se, se);
                    }
            } else {
#pragma unroll
                for (int j = 0; j < P; ++j) {
                    float2 ce = {1.f, 1.f}, se = {0.f, 0.f};
                    if (rot[i][0]) {
                        ce = *reinterpret_cast<const float2 *>(cos_row + off[i][0] + 2 * j);
                        se = *reinterpret_cast<const float2 *>(sin_row + off[i][0] + 2 * j);
                    }
                    c[i][0][j] = c[i][1][j] = f2(ce.x, ce.y);
                    s[i][0][j] = f2(-sign * se.x, -sign * se.y);
                    s[i][1][j] = f2(sign * se.x, sign * se.y);
                }
            }
        }
    }
    __device__ __forceinline__ void load_gains(const T *gamma, float g0, F2 (&g)[ITEMS][2][P]) const {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int v = 0; v < 2; ++v)
#pragma unroll
                for (int j = 0; j < P; ++j) {
                    g[i][v][j] = f2(0.f, 0.f);
                    if (off[i][v] >= 0) g[i][v][j] = f2(qk_to_f<T>(gamma[off[i][v] + 2 * j]) + g0, qk_to_f<T>(gamma[off[i][v] + 2 * j + 1]) + g0);
                }
    }
    __device__ __forceinline__ void store_zeros(T *head, bool inside) const {
        const F2 zero[P] = {};
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int v = 0; v < 2; ++v)
                if (inside && off[i][v] >= 0) qk_store<T, V>(head + off[i][v], zero);
    }
    // x * m + partner * n for the lane's item i; an element that is not rotated takes nothing of its partner (which may be infinite)
    __device__ __forceinline__ void turn(int i, const F2 (&x)[2][P], const F2 (&m)[2][P], const F2 (&n)[2][P], bool full, F2 (&y)[2][P]) const {
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
            for (int j = 0; j < P; ++j) {
                const F2 other = IL ? f2_swap(x[v][j]) : x[1 - v][j];
                const F2 own = f2_mul(x[v][j], m[v][j]);
                if (full) y[v][j] = f2_fma(other, n[v][j], own);
                else y[v][j] = rot[i][v] ? f2_fma(other, n[v][j], own) : own;
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
__global__ void __launch_bounds__(kQkThreads, kQkFwdCtas) qk_norm_rope_fwd_kernel(QkArgs a) {
    constexpr int kRows = 32 / G, P = V / 2;
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31;
    const uint32_t per_token = a.chunks[0] + a.chunks[1];
    const uint32_t unit = blockIdx.x * (kQkThreads / 32) + (threadIdx.x >> 5);
    const uint32_t t = unit / per_token;
    if (t >= a.T) return;
    int chunk = (int) (unit - t * per_token);
    const int r = chunk >= a.chunks[0];
    chunk -= r ? a.chunks[0] : 0;
    const uint32_t b = a.S == a.T ? 0 : t / (uint32_t) a.S, ti = t - b * (uint32_t) a.S;
    const int heads = a.heads[r], h0 = chunk * kRows * U + lane / G;
    const int64_t xh = a.xh[r];
    const T *x = reinterpret_cast<const T *>(a.x[r]) + b * a.xb[r] + ti * a.xt[r] + h0 * xh;
    const int64_t pos = qk_position(a, t, ti);   // first: the table's rows wait for it (62.7 us where 64.8 with the heads' loads before it)
    QkLane<T, V, G, ITEMS, IL> ln;
    ln.init(lane, a.D, a.R);

    QkWords<T, V> raw[U][ITEMS][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                raw[u][i][v] = QkWords<T, V>{};
                if (h0 + u * kRows < heads && ln.off[i][v] >= 0) raw[u][i][v] = qk_load<T, V>(x + u * kRows * xh + ln.off[i][v]);
            }
    T *out = reinterpret_cast<T *>(a.out[r]) + ((int64_t) t * heads + h0) * a.D;
    if (pos < 0) {   // the same for the whole warp
        for (int u = 0; u < U; ++u) ln.store_zeros(out + u * kRows * a.D, h0 + u * kRows < heads);
        return;
    }
    const bool full = a.R == a.D;
    F2 m[ITEMS][2][P], n[ITEMS][2][P];   // gain times cosine; the partner's gain times the signed sine
    {
        F2 c[ITEMS][2][P], s[ITEMS][2][P], g[ITEMS][2][P];
        const int64_t row = pos * (a.R / 2);
        ln.load_table(a.cos + row, a.sin + row, 1.f, c, s);
        ln.load_gains(reinterpret_cast<const T *>(a.gamma[r]), a.g0, g);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int v = 0; v < 2; ++v)
#pragma unroll
                for (int j = 0; j < P; ++j) {
                    m[i][v][j] = f2_mul(g[i][v][j], c[i][v][j]);
                    n[i][v][j] = f2_mul(IL ? f2_swap(g[i][v][j]) : g[i][1 - v][j], s[i][v][j]);
                }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        F2 xs[ITEMS][2][P], ss2 = f2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int v = 0; v < 2; ++v)
#pragma unroll
                for (int j = 0; j < P; ++j) {
                    xs[i][v][j] = qk_pair<T, V>(raw[u][i][v], j);
                    ss2 = f2_fma(xs[i][v][j], xs[i][v][j], ss2);
                }
        float rstd = rsqrtf(qk_group_sum<G>(f2_sum(ss2)) * a.inv_d + a.eps);
        const F2 scale = f2(rstd, rstd);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            F2 y[2][P];
            ln.turn(i, xs[i], m[i], n[i], full, y);
#pragma unroll
            for (int v = 0; v < 2; ++v) {
#pragma unroll
                for (int j = 0; j < P; ++j) y[v][j] = f2_mul(y[v][j], scale);
                if (h0 + u * kRows < heads && ln.off[i][v] >= 0) qk_store<T, V>(out + u * kRows * a.D + ln.off[i][v], y[v]);
            }
        }
    }
}

// Persistent CTAs: the first parts_q work on queries, the rest on keys, so that a lane's share of dgamma stays in registers over
// all its heads.  Per CTA one row of partial sums (fixed order: lanes, then warps); qk_dgamma_kernel adds the rows.
template <typename T, int V, int G, int ITEMS, bool IL, int U>
__global__ void __launch_bounds__(kQkBwdThreads, kQkBwdCtas) qk_norm_rope_bwd_kernel(QkArgs a) {
    constexpr int kRows = 32 / G, P = V / 2;
    constexpr int kWarps = kQkBwdThreads / 32;
    extern __shared__ float s_part[];   // [warps][D]
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r = (int) blockIdx.x >= a.parts_q;
    const uint32_t cta = blockIdx.x - (r ? a.parts_q : 0), ctas = r ? a.parts - a.parts_q : a.parts_q;
    const uint32_t chunks = a.chunks[r], units = (uint32_t) a.T * chunks;
    const int heads = a.heads[r];
    const int64_t xh = a.xh[r], gh = a.gh[r];
    const bool full = a.R == a.D;
    QkLane<T, V, G, ITEMS, IL> ln;
    ln.init(lane, a.D, a.R);
    F2 g[ITEMS][2][P], dg[ITEMS][2][P];
    ln.load_gains(reinterpret_cast<const T *>(a.gamma[r]), a.g0, g);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
            for (int j = 0; j < P; ++j) dg[i][v][j] = f2(0.f, 0.f);
    for (uint32_t unit = cta * kWarps + warp; unit < units; unit += ctas * kWarps) {
        const uint32_t t = unit / chunks, b = a.S == a.T ? 0 : t / (uint32_t) a.S, ti = t - b * (uint32_t) a.S;
        const int h0 = (int) (unit - t * chunks) * kRows * U + lane / G;
        const T *x = reinterpret_cast<const T *>(a.x[r]) + b * a.xb[r] + ti * a.xt[r] + h0 * xh;
        const T *dy = reinterpret_cast<const T *>(a.dy[r]) + b * a.gb[r] + ti * a.gt[r] + h0 * gh;
        const int64_t pos = qk_position(a, t, ti);
        QkWords<T, V> rx[U][ITEMS][2], rd[U][ITEMS][2];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    rx[u][i][v] = QkWords<T, V>{};
                    rd[u][i][v] = QkWords<T, V>{};
                    if (h0 + u * kRows < heads && ln.off[i][v] >= 0) {
                        rx[u][i][v] = qk_load<T, V>(x + u * kRows * xh + ln.off[i][v]);
                        rd[u][i][v] = qk_load<T, V>(dy + u * kRows * gh + ln.off[i][v]);
                    }
                }
        T *dx = reinterpret_cast<T *>(a.out[r]) + ((int64_t) t * heads + h0) * a.D;
        if (pos < 0) {   // the same for the whole warp; nothing for dgamma either
            for (int u = 0; u < U; ++u) ln.store_zeros(dx + u * kRows * a.D, h0 + u * kRows < heads);
            continue;
        }
        const int64_t row = pos * (a.R / 2);
        F2 c[ITEMS][2][P], s[ITEMS][2][P];
        ln.load_table(a.cos + row, a.sin + row, -1.f, c, s);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            F2 xs[ITEMS][2][P], dn[ITEMS][2][P], ss2 = f2(0.f, 0.f), dot2 = f2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                F2 d[2][P];
#pragma unroll
                for (int v = 0; v < 2; ++v)
#pragma unroll
                    for (int j = 0; j < P; ++j) {
                        xs[i][v][j] = qk_pair<T, V>(rx[u][i][v], j);
                        d[v][j] = qk_pair<T, V>(rd[u][i][v], j);
                        ss2 = f2_fma(xs[i][v][j], xs[i][v][j], ss2);
                    }
                ln.turn(i, d, c[i], s[i], full, dn[i]);
#pragma unroll
                for (int v = 0; v < 2; ++v)
#pragma unroll
                    for (int j = 0; j < P; ++j) dot2 = f2_fma(f2_mul(dn[i][v][j], g[i][v][j]), xs[i][v][j], dot2);
            }
            const float rstd = rsqrtf(qk_group_sum<G>(f2_sum(ss2)) * a.inv_d + a.eps);
            const float mean = qk_group_sum<G>(f2_sum(dot2)) * rstd * a.inv_d;   // mean(dn * g * xhat)
            if (h0 + u * kRows >= heads) continue;
            const F2 r2 = f2(rstd, rstd), m2 = f2(-mean * rstd, -mean * rstd);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    F2 o[P];
#pragma unroll
                    for (int j = 0; j < P; ++j) {
                        const F2 xhat = f2_mul(xs[i][v][j], r2);
                        o[j] = f2_fma(xhat, m2, f2_mul(f2_mul(dn[i][v][j], g[i][v][j]), r2));
                        dg[i][v][j] = f2_fma(dn[i][v][j], xhat, dg[i][v][j]);
                    }
                    if (ln.off[i][v] >= 0) qk_store<T, V>(dx + u * kRows * a.D + ln.off[i][v], o);
                }
        }
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
            for (int j = 0; j < P; ++j) {
                float d[2];
                f2_split(dg[i][v][j], d[0], d[1]);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int o = G; o < 32; o <<= 1) d[e] += __shfl_xor_sync(0xffffffffu, d[e], o);
                    if (lane < G && ln.off[i][v] >= 0) s_part[warp * a.D + ln.off[i][v] + 2 * j + e] = d[e];
                }
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
        const int64_t b = t / a.S, ti = t - b * a.S, pos = qk_position(a, (uint32_t) t, (uint32_t) ti);
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

// dgamma = sum of the partial rows of its side, in a fixed order; blockIdx.y: 0 queries, 1 keys.  A warp per 32 columns and every 32nd
// row, up to 16 rows in flight: one or two memory latencies (with 16 warps and 4 rows in flight this tail took 7 us).
constexpr int kDgWarps = 32;
template <typename T>
__global__ void __launch_bounds__(32 * kDgWarps) qk_dgamma_kernel(const float *__restrict__ partial, int parts_q, int parts, int D, T *dq_gamma,
                                                                  T *dk_gamma) {
    __shared__ float s_sum[kDgWarps][33];
    grid_dep_wait();
    const int c = threadIdx.x & 31, warp = threadIdx.x >> 5, d = (int) blockIdx.x * 32 + c;
    const int first = blockIdx.y ? parts_q : 0, last = blockIdx.y ? parts : parts_q;
    float acc = 0.f;
    if (d < D) {
        for (int p0 = first + warp; p0 < last; p0 += 16 * kDgWarps) {
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = p0 + i * kDgWarps < last ? partial[(int64_t) (p0 + i * kDgWarps) * D + d] : 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) acc += v[i];
        }
    }
    s_sum[warp][c] = acc;
    __syncthreads();
    if (warp == 0 && d < D) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < kDgWarps; ++i) t += s_sum[i][c];
        (blockIdx.y ? dk_gamma : dq_gamma)[d] = qk_from_f<T>(t);
    }
}

// ------------------------------------------------------------------------------------------------ host side
// How a head is laid over lanes: elements per access, four when the head, both halves of the rotation and every stride are whole
// vectors of them, else two; 0: the element-wise kernel.
static int qk_vec(const QkArgs &a, int esize, bool il, bool bwd) {
    for (int v : {4, 2}) {
        bool ok = aligned(a.cos, 8) && aligned(a.sin, 8) && a.D % v == 0 && (il ? a.R : a.R / 2) % v == 0 && a.R % v == 0;
        for (int r = 0; r < 2; ++r) {
            ok = ok && aligned(a.x[r], v * esize) && aligned(a.gamma[r], v * esize) && aligned(a.out[r], v * esize) &&
                 (a.xb[r] | a.xt[r] | a.xh[r]) % v == 0;
            if (bwd) ok = ok && aligned(a.dy[r], v * esize) && (a.gb[r] | a.gt[r] | a.gh[r]) % v == 0;
        }
        const int items = il ? (a.D / v + 1) / 2 : a.R / 2 / v + ((a.D - a.R) / v + 1) / 2;
        if (ok && items <= 64) return v;
    }
    return 0;
}

template <typename T, int V, int G, int ITEMS, bool IL> static int qk_launch(QkArgs a, bool bwd, cudaStream_t st) {
    // heads per lane group and warp, their loads in flight together; one where a token has fewer
    constexpr int kRows = 32 / G, kMost = (ITEMS == 1 ? 4 : 2) / (sizeof(T) == 4 ? 2 : 1);
    const int most = std::max(a.heads[0], a.heads[1]);
    auto set_chunks = [&](int U) { for (int r = 0; r < 2; ++r) a.chunks[r] = (int) ceil_div(a.heads[r], kRows * U); };
    if (!bwd) {
        auto go = [&](auto u) {
            constexpr int U = decltype(u)::value;
            set_chunks(U);
            const int64_t grid = ceil_div(a.T * (a.chunks[0] + a.chunks[1]), kQkThreads / 32);
            PT_CUDA_OK(launch_overlapped(qk_norm_rope_fwd_kernel<T, V, G, ITEMS, IL, U>, dim3((unsigned) grid), dim3(kQkThreads), 0, st, a));
            return (int) PT_OK;
        };
        return most >= 2 * kRows ? go(std::integral_constant<int, kMost>{}) : go(std::integral_constant<int, 1>{});
    }
    constexpr int U = ITEMS == 1 && sizeof(T) == 2 ? 2 : 1;
    set_chunks(U);
    PT_CUDA_OK(launch_overlapped(qk_norm_rope_bwd_kernel<T, V, G, ITEMS, IL, U>, dim3(a.parts), dim3(kQkBwdThreads),
                                 (size_t) (kQkBwdThreads / 32) * a.D * 4, st, a));
    return PT_OK;
}

template <typename T, bool IL> static int qk_dispatch(const QkArgs &a, bool bwd, cudaStream_t st) {
    const int v = qk_vec(a, sizeof(T), IL, bwd);
    if (v == 0) {
        const size_t smem = bwd ? (size_t) (kQkBwdThreads / 32) * a.D * 4 : 0;
        const int64_t fwd_grid = std::min<int64_t>(ceil_div(a.T * (a.heads[0] + a.heads[1]), kQkBwdThreads / 32), (int64_t) sm_count() * 8);
        if (bwd) PT_CUDA_OK(launch_overlapped(qk_norm_rope_any_kernel<T, true>, dim3(a.parts), dim3(kQkBwdThreads), smem, st, a, (int) IL));
        else PT_CUDA_OK(launch_overlapped(qk_norm_rope_any_kernel<T, false>, dim3((unsigned) fwd_grid), dim3(kQkBwdThreads), smem, st, a, (int) IL));
        return PT_OK;
    }
    const int items = IL ? (a.D / v + 1) / 2 : a.R / 2 / v + ((a.D - a.R) / v + 1) / 2;
    if (v == 4) {
        if (items <= 8) return qk_launch<T, 4, 8, 1, IL>(a, bwd, st);
        if (items <= 16) return qk_launch<T, 4, 16, 1, IL>(a, bwd, st);
        if (items <= 32) return qk_launch<T, 4, 32, 1, IL>(a, bwd, st);
        return qk_launch<T, 4, 32, 2, IL>(a, bwd, st);
    }
    if (items <= 16) return qk_launch<T, 2, 16, 1, IL>(a, bwd, st);
    if (items <= 32) return qk_launch<T, 2, 32, 1, IL>(a, bwd, st);
    return qk_launch<T, 2, 32, 2, IL>(a, bwd, st);
}

// Host strides (batch, token, head) into the arguments; the stride of an extent of one is never used, but would decide the
// alignment of the vector accesses, so it counts as zero.
static void qk_strides(const int64_t *s, int64_t B, int64_t S, int heads, int64_t &b, int64_t &t, int64_t &h) {
    b = B > 1 ? s[0] : 0;
    t = S > 1 ? s[1] : 0;
    h = heads > 1 ? s[2] : 0;
}

static int qk_check(const QkArgs &a, int dtype, int64_t B) {
    PT_REQUIRE(dtype == PT_BF16 || dtype == PT_F16 || dtype == PT_F32, "qk_norm_rope: unsupported dtype %d", dtype);
    PT_REQUIRE(B >= 0 && a.S >= 0 && a.heads[0] >= 0 && a.heads[1] >= 0, "qk_norm_rope: negative extent");
    PT_REQUIRE(a.D >= 1 && a.D <= kQkMaxD && a.R >= 0 && a.R % 2 == 0 && a.R <= a.D,
               "qk_norm_rope: the head size must lie in [1, %d] and the rotated part be even and no larger (got %d, %d)", kQkMaxD, a.D, a.R);
    PT_REQUIRE(a.T < (1ll << 31) && a.T * (a.heads[0] + (int64_t) a.heads[1]) < (1ll << 31), "qk_norm_rope: tokens x heads exceed 32-bit indices");
    PT_REQUIRE(a.pos_bytes == 0 || a.pos_bytes == 4 || a.pos_bytes == 8, "qk_norm_rope: positions must be int32 or int64");
    // an empty tensor is a null pointer
    PT_REQUIRE(a.T == 0 || (a.pos_bytes == 0) == (a.positions == nullptr), "qk_norm_rope: positions and their size go together");
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
    qk_strides(q_strides, B, S, Hq, a.xb[0], a.xt[0], a.xh[0]);
    qk_strides(k_strides, B, S, Hk, a.xb[1], a.xt[1], a.xh[1]);
    a.heads[0] = Hq; a.heads[1] = Hk; a.cos = cos; a.sin = sin; a.positions = positions; a.pos_bytes = pos_bytes;
    a.T = B * S; a.S = S; a.P = P; a.D = D; a.R = R; a.eps = eps; a.inv_d = 1.f / (float) std::max(D, 1); a.g0 = zero_centered ? 1.f : 0.f;
    a.status = status;
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
    qk_strides(q_strides, B, S, Hq, a.xb[0], a.xt[0], a.xh[0]);
    qk_strides(k_strides, B, S, Hk, a.xb[1], a.xt[1], a.xh[1]);
    qk_strides(dq_strides, B, S, Hq, a.gb[0], a.gt[0], a.gh[0]);
    qk_strides(dk_strides, B, S, Hk, a.gb[1], a.gt[1], a.gh[1]);
    a.heads[0] = Hq; a.heads[1] = Hk; a.cos = cos; a.sin = sin; a.positions = positions; a.pos_bytes = pos_bytes;
    a.T = B * S; a.S = std::max<int64_t>(S, 1); a.P = P; a.D = D; a.R = R; a.eps = eps; a.inv_d = 1.f / (float) std::max(D, 1);
    a.g0 = zero_centered ? 1.f : 0.f; a.status = status;
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
        PT_CUDA_OK(launch_overlapped(qk_dgamma_kernel<T>, dim3((unsigned) ceil_div(D, 32), 2), dim3(32 * kDgWarps), 0, st, (const float *) partial, a.parts_q, a.parts, D,
                                     (T *) dq_gamma, (T *) dk_gamma));
    });
    return PT_OK;
}

}  // extern "C"
