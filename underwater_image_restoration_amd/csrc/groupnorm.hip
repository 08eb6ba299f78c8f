// Group norm with an activation on NHWC rows, forward and backward.
//   mean, var over the n x cg elements of (image, group);  xh = (x - mean) rstd
//   z = (xh gamma + beta)(1 + scale_b) + shift_b;   y = act(z),  act = identity or SiLU
// Both directions are bound by memory (or, for small maps, by launch latency).  Two forms:
//   resident  a block owns a slab of whole groups of one image, keeps its rows in registers between the statistics and
//             the output, and so touches every element once (one launch);
//   streamed  statistics of row chunks in one launch, output in the next; the second read of x comes from the L2 / the
//             memory-side cache where the map fits.
// Statistics: every thread reduces batches of rows to (mean, sum of squared distances to that mean) per channel and
// merges them pairwise, so that a mean far from zero or a stray first element costs no digits; everything across
// threads is summed in fp64 in a fixed order (results do not depend on scheduling).
#include "common.h"
#include <type_traits>

namespace {

constexpr int GN_T = 256;          // threads of the streaming kernels
constexpr int GN_R = 8;            // rows a thread loads ahead of using them
constexpr int GN_MAX_C = 2048;     // per-channel fp64 sums of one block live in LDS
constexpr int GN_MAX_CHUNKS = 128; // row chunks of an image (each output block sums all of an image's partials)

template <typename T, int V> struct VecT { typedef T type __attribute__((ext_vector_type(V))); };
template <typename T> struct VecT<T, 1> { typedef T type; };

template <typename T, int V> struct Pack {
    typename VecT<T, V>::type v;
    __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const typename VecT<T, V>::type*>(p); }
    __device__ __forceinline__ float get(int j) const {
        if constexpr (V == 1) return (float)v;
        else return (float)v[j];
    }
    __device__ __forceinline__ void set(int j, float f) {
        if constexpr (V == 1) v = (T)f;
        else v[j] = (T)f;
    }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<typename VecT<T, V>::type*>(p) = v; }
};

struct GnArgs {
    const void *x, *dy;
    void* out;                       // y, or dx
    const float *gamma, *beta, *ss;  // ss [B, ld_ss]: [scale | shift], or NULL
    const float *mean_in, *rstd_in;  // backward
    float *mean, *rstd;              // forward, optional
    float *dgamma, *dbeta, *dss;     // backward; dss [B, ld_dss] optional
    double2* part;                   // forward partials [B][chunks][G]: (sum, sum of squares)
    float2* cpart;                   // backward partials [B][chunks][C]: (sum dz, sum dz xh)
    float2* csum;                    // backward [B][C]
    size_t ldx, ldy, ldo, ld_ss, ld_dss;
    int B, n, C, G, cg, chunks, rows, slab;  // rows per chunk; channels per slab
    float eps;
    int act;
};

// per-channel running statistics of one thread: V channels, `cnt` rows so far
template <int V> struct Stat {
    float mean[V], m2[V];
    int cnt;
    __device__ __forceinline__ void clear() {
        cnt = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) mean[j] = m2[j] = 0.f;
    }
    // merge `k` <= GN_R fresh rows (pairwise update: exact in the count weights)
    template <typename T> __device__ __forceinline__ void batch(const Pack<T, V>* p, int k) {
        if (k <= 0) return;
        const float inv = 1.f / (float)k;
        const float wa = (float)k / (float)(cnt + k), wb = (float)cnt * wa;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < GN_R; ++i) s += i < k ? p[i].get(j) : 0.f;
            const float m = s * inv;
            float q = 0.f;
#pragma unroll
            for (int i = 0; i < GN_R; ++i) {
                const float d = i < k ? p[i].get(j) - m : 0.f;
                q = fmaf(d, d, q);
            }
            const float d = m - mean[j];
            mean[j] = fmaf(d, wa, mean[j]);
            m2[j] += fmaf(d * d, wb, q);
        }
        cnt += k;
    }
};

__device__ __forceinline__ double shfl_xor_d(double v, int m) {
    return __hiloint2double(__shfl_xor(__double2hiint(v), m), __shfl_xor(__double2loint(v), m));
}

// threads that share one group's reduction: a power of two <= 64 with tpg * G <= T where that is possible
__device__ __forceinline__ int threads_per_group(int G, int T) {
    int t = 64;
    while (t > 1 && t * G > T) t >>= 1;
    return t;
}

// sums over groups of f(g, i) for i in [0, m): result in every lane of the group's team, handed to `done(g, a, b)` by lane 0
template <typename F, typename D>
__device__ __forceinline__ void group_sums(int G, int m, int tid, int T, F f, D done) {
    const int tpg = threads_per_group(G, T), teams = T / tpg, lane = tid & (tpg - 1);
    for (int g0 = 0; g0 < G; g0 += teams) {   // uniform trip count: the shuffles below see whole waves
        const int g = g0 + tid / tpg;
        double a = 0., b = 0.;
        if (g < G)
            for (int i = lane; i < m; i += tpg) {
                const double2 v = f(g, i);
                a += v.x;
                b += v.y;
            }
        for (int o = tpg >> 1; o; o >>= 1) {
            a += shfl_xor_d(a, o);
            b += shfl_xor_d(b, o);
        }
        if (g < G && lane == 0) done(g, a, b);
    }
}

__device__ __forceinline__ float act_silu(float z) { return z * sigmoid_fast(z); }
__device__ __forceinline__ float dact_silu(float z) {
    const float s = sigmoid_fast(z);
    return s * fmaf(z, 1.f - s, 1.f);
}

// ---------------------------------------------------------------------------------------- forward, streamed
template <typename TX, int V>
__global__ void __launch_bounds__(GN_T) gn_stats_kernel(GnArgs p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float* sm = reinterpret_cast<float*>(smem);                        // [GN_T][V] means
    float* sq = sm + GN_T * V;                                         // [GN_T][V] squares
    double2* ch = reinterpret_cast<double2*>(sq + GN_T * V);           // [C] (sum, sum of squares)
    const int tid = threadIdx.x, chunk = blockIdx.x, b = blockIdx.y;
    const int nv = p.C / V;
    const int r0 = chunk * p.rows, r1 = min(p.n, r0 + p.rows);
    const TX* X = (const TX*)p.x + (size_t)b * p.n * p.ldx;
    for (int c0 = 0; c0 < nv; c0 += GN_T) {
        const int tw = min(nv - c0, GN_T), RL = GN_T / tw, cv = tid % tw, rl = tid / tw;
        Stat<V> st;
        st.clear();
        if (rl < RL) {
            const TX* src = X + (size_t)(c0 + cv) * V;
            for (int r = r0 + rl; r < r1; r += RL * GN_R) {
                Pack<TX, V> buf[GN_R];
                const int k = min(GN_R, (r1 - r + RL - 1) / RL);
#pragma unroll
                for (int i = 0; i < GN_R; ++i) buf[i].load(src + (size_t)(i < k ? r + i * RL : r) * p.ldx);
                st.batch(buf, k);
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            sm[tid * V + j] = st.mean[j];
            sq[tid * V + j] = st.m2[j];
        }
        __syncthreads();
        for (int c = tid; c < tw * V; c += GN_T) {
            double s = 0., q = 0.;
            for (int l = 0; l < RL; ++l) {
                const int left = r1 - r0 - l;
                const double k = left > 0 ? (left + RL - 1) / RL : 0;
                const double m = sm[l * tw * V + c];
                s += k * m;
                q += sq[l * tw * V + c] + k * m * m;
            }
            ch[c0 * V + c] = make_double2(s, q);
        }
        __syncthreads();
    }
    double2* out = p.part + ((size_t)b * p.chunks + chunk) * p.G;
    const int cg = p.cg;
    group_sums(p.G, cg, tid, GN_T, [&](int g, int i) { return ch[g * cg + i]; },
               [&](int g, double s, double q) { out[g] = make_double2(s, q); });
}

__device__ __forceinline__ float2 finish_stats(double s, double q, double N, float eps) {
    const double m = s / N;
    double v = q / N - m * m;
    v = v > 0. ? v : 0.;
    return make_float2((float)m, (float)(1. / sqrt(v + (double)eps)));
}

// folded per-channel coefficients: z = (x - m) a + s
__device__ __forceinline__ void channel_affine(const GnArgs& p, int b, int c, float rstd, float& a, float& s) {
    const float ga = p.gamma[c], be = p.beta[c];
    float f = 1.f, sh = 0.f;
    if (p.ss) {
        f = 1.f + p.ss[(size_t)b * p.ld_ss + c];
        sh = p.ss[(size_t)b * p.ld_ss + p.C + c];
    }
    a = rstd * ga * f;
    s = fmaf(be, f, sh);
}

template <typename TX, typename TO, int V>
__global__ void __launch_bounds__(GN_T) gn_apply_kernel(GnArgs p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float2* gst = reinterpret_cast<float2*>(smem);   // [G] (mean, rstd)
    const int tid = threadIdx.x, chunk = blockIdx.x, b = blockIdx.y;
    const int nv = p.C / V, cg = p.cg;
    const double2* part = p.part + (size_t)b * p.chunks * p.G;
    const double N = (double)p.n * cg;
    group_sums(p.G, p.chunks, tid, GN_T, [&](int g, int i) { return part[(size_t)i * p.G + g]; },
               [&](int g, double s, double q) {
                   const float2 st = finish_stats(s, q, N, p.eps);
                   gst[g] = st;
                   if (chunk == 0) {
                       if (p.mean) p.mean[(size_t)b * p.G + g] = st.x;
                       if (p.rstd) p.rstd[(size_t)b * p.G + g] = st.y;
                   }
               });
    __syncthreads();
    const int r0 = chunk * p.rows, r1 = min(p.n, r0 + p.rows);
    const TX* X = (const TX*)p.x + (size_t)b * p.n * p.ldx;
    TO* Y = (TO*)p.out + (size_t)b * p.n * p.ldo;
    const bool silu = p.act == UWIR_ACT_SILU;
    for (int c0 = 0; c0 < nv; c0 += GN_T) {
        const int tw = min(nv - c0, GN_T), RL = GN_T / tw, cv = tid % tw, rl = tid / tw;
        if (rl >= RL) continue;
        const int cb = (c0 + cv) * V;
        float m[V], a[V], s[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float2 st = gst[(cb + j) / cg];
            m[j] = st.x;
            channel_affine(p, b, cb + j, st.y, a[j], s[j]);
        }
        for (int r = r0 + rl; r < r1; r += RL * GN_R) {
            Pack<TX, V> buf[GN_R];
            const int k = min(GN_R, (r1 - r + RL - 1) / RL);
#pragma unroll
            for (int i = 0; i < GN_R; ++i) buf[i].load(X + (size_t)(i < k ? r + i * RL : r) * p.ldx + cb);
#pragma unroll
            for (int i = 0; i < GN_R; ++i)
                if (i < k) {
                    Pack<TO, V> o;
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float z = fmaf(buf[i].get(j) - m[j], a[j], s[j]);
                        o.set(j, silu ? act_silu(z) : z);
                    }
                    o.store(Y + (size_t)(r + i * RL) * p.ldo + cb);
                }
        }
    }
}

// ---------------------------------------------------------------------------------------- forward, resident
template <typename TX, typename TO, int V, int T>
__global__ void __launch_bounds__(T) gn_resident_kernel(GnArgs p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float* sm = reinterpret_cast<float*>(smem);
    float* sq = sm + T * V;
    double2* ch = reinterpret_cast<double2*>(sq + T * V);              // [slab]
    float2* gst = reinterpret_cast<float2*>(ch + p.slab);              // [slab / cg]
    const int tid = threadIdx.x, b = blockIdx.y, cg = p.cg;
    const int ch0 = blockIdx.x * p.slab, sc = min(p.slab, p.C - ch0), gs = sc / cg, g0 = ch0 / cg;
    const int tw = sc / V, RL = T / tw, cv = tid % tw, rl = tid / tw;
    const TX* X = (const TX*)p.x + (size_t)b * p.n * p.ldx + ch0 + cv * V;
    Pack<TX, V> buf[GN_R];
    const int k = rl < RL && rl < p.n ? (p.n - rl + RL - 1) / RL : 0;  // <= GN_R by the launch rule
    if (k > 0) {
#pragma unroll
        for (int i = 0; i < GN_R; ++i) buf[i].load(X + (size_t)(i < k ? rl + i * RL : rl) * p.ldx);
    }
    Stat<V> st;
    st.clear();
    st.batch(buf, k);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        sm[tid * V + j] = st.mean[j];
        sq[tid * V + j] = st.m2[j];
    }
    __syncthreads();
    const int rows = min(RL, p.n);
    for (int c = tid; c < sc; c += T) {
        double s = 0., q = 0.;
        for (int l = 0; l < rows; ++l) {
            const double kk = (p.n - l + RL - 1) / RL, m = sm[l * sc + c];
            s += kk * m;
            q += sq[l * sc + c] + kk * m * m;
        }
        ch[c] = make_double2(s, q);
    }
    __syncthreads();
    const double N = (double)p.n * cg;
    group_sums(gs, cg, tid, T, [&](int g, int i) { return ch[g * cg + i]; },
               [&](int g, double s, double q) {
                   const float2 f = finish_stats(s, q, N, p.eps);
                   gst[g] = f;
                   if (p.mean) p.mean[(size_t)b * p.G + g0 + g] = f.x;
                   if (p.rstd) p.rstd[(size_t)b * p.G + g0 + g] = f.y;
               });
    __syncthreads();
    if (k <= 0) return;
    const bool silu = p.act == UWIR_ACT_SILU;
    float m[V], a[V], s[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float2 f = gst[(cv * V + j) / cg];
        m[j] = f.x;
        channel_affine(p, b, ch0 + cv * V + j, f.y, a[j], s[j]);
    }
    TO* Y = (TO*)p.out + (size_t)b * p.n * p.ldo + ch0 + cv * V;
#pragma unroll
    for (int i = 0; i < GN_R; ++i)
        if (i < k) {
            Pack<TO, V> o;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float z = fmaf(buf[i].get(j) - m[j], a[j], s[j]);
                o.set(j, silu ? act_silu(z) : z);
            }
            o.store(Y + (size_t)(rl + i * RL) * p.ldo);
        }
}

// ---------------------------------------------------------------------------------------- backward, streamed
// per-channel coefficients of a thread: z = (x - m) a + s, xh = (x - m) r
template <int V> struct BwdCoef {
    float m[V], r[V], a[V], s[V];
    __device__ __forceinline__ void load(const GnArgs& p, int b, int c0) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = c0 + j, g = c / p.cg;
            m[j] = p.mean_in[(size_t)b * p.G + g];
            r[j] = p.rstd_in[(size_t)b * p.G + g];
            channel_affine(p, b, c, r[j], a[j], s[j]);
        }
    }
    __device__ __forceinline__ void grad(int j, float x, float dy, bool silu, float& dz, float& xh) const {
        const float d = x - m[j];
        xh = d * r[j];
        dz = silu ? dy * dact_silu(fmaf(d, a[j], s[j])) : dy;
    }
};

template <typename T, int V>
__global__ void __launch_bounds__(GN_T) gn_bwd_sums_kernel(GnArgs p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float2* red = reinterpret_cast<float2*>(smem);   // [GN_T][V]
    const int tid = threadIdx.x, chunk = blockIdx.x, b = blockIdx.y;
    const int nv = p.C / V;
    const int r0 = chunk * p.rows, r1 = min(p.n, r0 + p.rows);
    const T* X = (const T*)p.x + (size_t)b * p.n * p.ldx;
    const T* DY = (const T*)p.dy + (size_t)b * p.n * p.ldy;
    float2* out = p.cpart + ((size_t)b * p.chunks + chunk) * p.C;
    const bool silu = p.act == UWIR_ACT_SILU;
    constexpr int R = GN_R / 2;
    for (int c0 = 0; c0 < nv; c0 += GN_T) {
        const int tw = min(nv - c0, GN_T), RL = GN_T / tw, cv = tid % tw, rl = tid / tw;
        const int cb = (c0 + cv) * V;
        float s1[V], s2[V];
#pragma unroll
        for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.f;
        if (rl < RL) {
            BwdCoef<V> co;
            co.load(p, b, cb);
            for (int r = r0 + rl; r < r1; r += RL * R) {
                Pack<T, V> bx[R], bd[R];
                const int k = min(R, (r1 - r + RL - 1) / RL);
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const size_t row = i < k ? r + i * RL : r;
                    bx[i].load(X + row * p.ldx + cb);
                    bd[i].load(DY + row * p.ldy + cb);
                }
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    float t1 = 0.f, t2 = 0.f;   // a short chain per batch keeps the fp32 sums close to pairwise
#pragma unroll
                    for (int i = 0; i < R; ++i)
                        if (i < k) {
                            float dz, xh;
                            co.grad(j, bx[i].get(j), bd[i].get(j), silu, dz, xh);
                            t1 += dz;
                            t2 = fmaf(dz, xh, t2);
                        }
                    s1[j] += t1;
                    s2[j] += t2;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) red[tid * V + j] = make_float2(s1[j], s2[j]);
        __syncthreads();
        for (int c = tid; c < tw * V; c += GN_T) {
            double a = 0., q = 0.;
            for (int l = 0; l < RL; ++l) {
                const float2 v = red[l * tw * V + c];
                a += v.x;
                q += v.y;
            }
            out[c0 * V + c] = make_float2((float)a, (float)q);
        }
        __syncthreads();
    }
}

// S1, S2 of 64 channels of one image: 4 lanes a channel over the chunks; the modulation's gradient falls out here
__global__ void __launch_bounds__(GN_T) gn_bwd_reduce_kernel(GnArgs p) {
    __shared__ double2 red[4][64];
    const int cl = threadIdx.x & 63, l = threadIdx.x >> 6, c = blockIdx.x * 64 + cl, b = blockIdx.y;
    double a = 0., q = 0.;
    if (c < p.C)
        for (int i = l; i < p.chunks; i += 4) {
            const float2 v = p.cpart[((size_t)b * p.chunks + i) * p.C + c];
            a += v.x;
            q += v.y;
        }
    red[l][cl] = make_double2(a, q);
    __syncthreads();
    if (l == 0 && c < p.C) {
        for (int i = 1; i < 4; ++i) {
            a += red[i][cl].x;
            q += red[i][cl].y;
        }
        p.csum[(size_t)b * p.C + c] = make_float2((float)a, (float)q);
        if (p.dss) {
            p.dss[(size_t)b * p.ld_dss + c] = (float)(p.gamma[c] * q + p.beta[c] * a);
            p.dss[(size_t)b * p.ld_dss + p.C + c] = (float)a;
        }
    }
}

// dgamma, dbeta of 64 channels: 4 lanes a channel over the images
__device__ __forceinline__ void affine_grads(const GnArgs& p, int tile, double2 (*red)[64]) {
    const int cl = threadIdx.x & 63, l = threadIdx.x >> 6, c = tile * 64 + cl;
    double dg = 0., db = 0.;
    if (c < p.C)
        for (int b = l; b < p.B; b += 4) {
            const float2 v = p.csum[(size_t)b * p.C + c];
            const double f = p.ss ? 1. + (double)p.ss[(size_t)b * p.ld_ss + c] : 1.;
            dg += f * v.y;
            db += f * v.x;
        }
    red[l][cl] = make_double2(dg, db);
    __syncthreads();
    if (l == 0 && c < p.C) {
        for (int i = 1; i < 4; ++i) {
            dg += red[i][cl].x;
            db += red[i][cl].y;
        }
        p.dgamma[c] = (float)dg;
        p.dbeta[c] = (float)db;
    }
}

__global__ void __launch_bounds__(GN_T) gn_bwd_affine_kernel(GnArgs p) {
    __shared__ double2 red[4][64];
    affine_grads(p, blockIdx.x, red);
}

// dx = r (w dz - m1 - xh m2); the last row of blocks (b == B) forms dgamma, dbeta instead
template <typename T, int V>
__global__ void __launch_bounds__(GN_T) gn_bwd_apply_kernel(GnArgs p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, chunk = blockIdx.x, b = blockIdx.y;
    if (b == p.B) {
        for (int t = chunk; t * 64 < p.C; t += gridDim.x) {
            affine_grads(p, t, reinterpret_cast<double2(*)[64]>(smem));
            __syncthreads();
        }
        return;
    }
    float2* gm = reinterpret_cast<float2*>(smem);   // [G] (m1, m2)
    const int nv = p.C / V, cg = p.cg;
    const double N = (double)p.n * cg;
    group_sums(p.G, cg, tid, GN_T,
               [&](int g, int i) {
                   const int c = g * cg + i;
                   const float2 v = p.csum[(size_t)b * p.C + c];
                   const double w = (double)p.gamma[c] * (p.ss ? 1. + (double)p.ss[(size_t)b * p.ld_ss + c] : 1.);
                   return make_double2(w * v.x, w * v.y);
               },
               [&](int g, double s, double q) { gm[g] = make_float2((float)(s / N), (float)(q / N)); });
    __syncthreads();
    const int r0 = chunk * p.rows, r1 = min(p.n, r0 + p.rows);
    const T* X = (const T*)p.x + (size_t)b * p.n * p.ldx;
    const T* DY = (const T*)p.dy + (size_t)b * p.n * p.ldy;
    T* DX = (T*)p.out + (size_t)b * p.n * p.ldo;
    const bool silu = p.act == UWIR_ACT_SILU;
    constexpr int R = GN_R / 2;
    for (int c0 = 0; c0 < nv; c0 += GN_T) {
        const int tw = min(nv - c0, GN_T), RL = GN_T / tw, cv = tid % tw, rl = tid / tw;
        if (rl >= RL) continue;
        const int cb = (c0 + cv) * V;
        BwdCoef<V> co;
        co.load(p, b, cb);
        float m1[V], m2[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float2 g = gm[(cb + j) / cg];
            m1[j] = co.r[j] * g.x;
            m2[j] = co.r[j] * g.y;
        }
        for (int r = r0 + rl; r < r1; r += RL * R) {
            Pack<T, V> bx[R], bd[R];
            const int k = min(R, (r1 - r + RL - 1) / RL);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const size_t row = i < k ? r + i * RL : r;
                bx[i].load(X + row * p.ldx + cb);
                bd[i].load(DY + row * p.ldy + cb);
            }
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (i < k) {
                    Pack<T, V> o;
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        float dz, xh;
                        co.grad(j, bx[i].get(j), bd[i].get(j), silu, dz, xh);
                        o.set(j, fmaf(co.a[j], dz, -fmaf(xh, m2[j], m1[j])));   // a = r w
                    }
                    o.store(DX + (size_t)(r + i * RL) * p.ldo + cb);
                }
        }
    }
}

// ---------------------------------------------------------------------------------------- backward, resident
template <typename T, int V, int TH>
__global__ void __launch_bounds__(TH) gn_bwd_resident_kernel(GnArgs p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float2* red = reinterpret_cast<float2*>(smem);                     // [TH][V]
    double2* ch = reinterpret_cast<double2*>(red + TH * V);            // [slab] w (S1, S2)
    float2* gm = reinterpret_cast<float2*>(ch + p.slab);               // [slab / cg]
    const int tid = threadIdx.x, b = blockIdx.y, cg = p.cg;
    const int ch0 = blockIdx.x * p.slab, sc = min(p.slab, p.C - ch0), gs = sc / cg;
    const int tw = sc / V, RL = TH / tw, cv = tid % tw, rl = tid / tw, cb = ch0 + cv * V;
    const T* X = (const T*)p.x + (size_t)b * p.n * p.ldx + cb;
    const T* DY = (const T*)p.dy + (size_t)b * p.n * p.ldy + cb;
    const bool silu = p.act == UWIR_ACT_SILU;
    const int k = rl < RL && rl < p.n ? (p.n - rl + RL - 1) / RL : 0;
    Pack<T, V> bx[GN_R], bd[GN_R];
    BwdCoef<V> co;
    float s1[V], s2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.f;
    if (k > 0) {
#pragma unroll
        for (int i = 0; i < GN_R; ++i) {
            const size_t row = i < k ? rl + i * RL : rl;
            bx[i].load(X + row * p.ldx);
            bd[i].load(DY + row * p.ldy);
        }
        co.load(p, b, cb);
#pragma unroll
        for (int i = 0; i < GN_R; ++i)
            if (i < k) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    float dz, xh;
                    co.grad(j, bx[i].get(j), bd[i].get(j), silu, dz, xh);
                    s1[j] += dz;
                    s2[j] = fmaf(dz, xh, s2[j]);
                }
            }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) red[tid * V + j] = make_float2(s1[j], s2[j]);
    __syncthreads();
    const int rows = min(RL, p.n);
    for (int c = tid; c < sc; c += TH) {
        double a = 0., q = 0.;
        for (int l = 0; l < rows; ++l) {
            const float2 v = red[l * sc + c];
            a += v.x;
            q += v.y;
        }
        const int cc = ch0 + c;
        const double ga = p.gamma[cc], f = p.ss ? 1. + (double)p.ss[(size_t)b * p.ld_ss + cc] : 1.;
        ch[c] = make_double2(ga * f * a, ga * f * q);
        if (p.dss) {
            p.dss[(size_t)b * p.ld_dss + cc] = (float)(ga * q + p.beta[cc] * a);
            p.dss[(size_t)b * p.ld_dss + p.C + cc] = (float)a;
        }
        if (p.B == 1) {   // nothing to sum over: the affine's gradient is complete
            p.dgamma[cc] = (float)(f * q);
            p.dbeta[cc] = (float)(f * a);
        } else {
            p.csum[(size_t)b * p.C + cc] = make_float2((float)a, (float)q);
        }
    }
    __syncthreads();
    const double N = (double)p.n * cg;
    group_sums(gs, cg, tid, TH, [&](int g, int i) { return ch[g * cg + i]; },
               [&](int g, double s, double q) { gm[g] = make_float2((float)(s / N), (float)(q / N)); });
    __syncthreads();
    if (k <= 0) return;
    T* DX = (T*)p.out + (size_t)b * p.n * p.ldo + cb;
    float m1[V], m2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float2 g = gm[(cv * V + j) / cg];
        m1[j] = co.r[j] * g.x;
        m2[j] = co.r[j] * g.y;
    }
#pragma unroll
    for (int i = 0; i < GN_R; ++i)
        if (i < k) {
            Pack<T, V> o;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float dz, xh;
                co.grad(j, bx[i].get(j), bd[i].get(j), silu, dz, xh);
                o.set(j, fmaf(co.a[j], dz, -fmaf(xh, m2[j], m1[j])));
            }
            o.store(DX + (size_t)(rl + i * RL) * p.ldo);
        }
}

// ---------------------------------------------------------------------------------------- launch rules
int gcd_i(int a, int b) { return b ? gcd_i(b, a % b) : a; }

// channels a block of the resident form owns: whole groups and whole vectors, at least 64 bytes of a row
int slab_channels(int C, int cg, int V, int es) {
    const int unit = cg / gcd_i(cg, V) * V;
    int s = unit;
    while (s * es < 64 && s < C) s += unit;
    return s < C ? s : C;
}

size_t resident_lds(int T, int slab, int cg, int V) { return (size_t)T * V * 8 + (size_t)slab * 16 + (size_t)(slab / cg) * 8; }

// threads of the resident form (0: the slab's rows do not fit the registers of a block, or its sums 64 KB of LDS)
int resident_threads(int n, int slab, int cg, int V) {
    const int tw = slab / V;
    for (int T = 256; T <= 512; T *= 2)
        if (tw <= T && (long long)(T / tw) * GN_R >= n && resident_lds(T, slab, cg, V) <= 65536) return T;
    return 0;
}

int stream_chunks(int B, int n) {
    int c = 1024 / (B > 0 ? B : 1);
    c = c < 1 ? 1 : (c > GN_MAX_CHUNKS ? GN_MAX_CHUNKS : c);
    const int most = ceil_div(n, 8);   // a chunk has a batch of rows at least
    return c < most ? c : most;
}

size_t al256(size_t v) { return (v + 255) & ~(size_t)255; }

bool vec_ok(const void* p, size_t ld, int V, int es) {
    const size_t a = (size_t)V * es > 16 ? 16 : (size_t)V * es;
    return ((uintptr_t)p % a) == 0 && (ld * es) % a == 0;
}

template <typename F> int with_v(int V, F f) {
    switch (V) {
        case 8: return f(std::integral_constant<int, 8>());
        case 4: return f(std::integral_constant<int, 4>());
        case 2: return f(std::integral_constant<int, 2>());
        default: return f(std::integral_constant<int, 1>());
    }
}

template <typename TX, typename TO, int V> void launch_fwd(GnArgs p, hipStream_t st) {
    const int es = sizeof(TX);
    p.slab = slab_channels(p.C, p.cg, V, es);
    const int T = resident_threads(p.n, p.slab, p.cg, V);
    if (T) {
        const size_t lds = resident_lds(T, p.slab, p.cg, V);
        const dim3 grid(ceil_div(p.C, p.slab), p.B);
        if (T == 256)
            hipLaunchKernelGGL((gn_resident_kernel<TX, TO, V, 256>), grid, dim3(256), lds, st, p);
        else
            hipLaunchKernelGGL((gn_resident_kernel<TX, TO, V, 512>), grid, dim3(512), lds, st, p);
        return;
    }
    p.chunks = stream_chunks(p.B, p.n);
    p.rows = ceil_div(p.n, p.chunks);
    const dim3 grid(p.chunks, p.B);
    hipLaunchKernelGGL((gn_stats_kernel<TX, V>), grid, dim3(GN_T), (size_t)GN_T * V * 8 + (size_t)p.C * 16, st, p);
    hipLaunchKernelGGL((gn_apply_kernel<TX, TO, V>), grid, dim3(GN_T), (size_t)p.G * 8, st, p);
}

template <typename T, int V> void launch_bwd(GnArgs p, hipStream_t st) {
    p.slab = slab_channels(p.C, p.cg, V, sizeof(T));
    const int TH = resident_threads(p.n, p.slab, p.cg, V);
    if (TH) {
        const size_t lds = resident_lds(TH, p.slab, p.cg, V);
        const dim3 grid(ceil_div(p.C, p.slab), p.B);
        if (TH == 256)
            hipLaunchKernelGGL((gn_bwd_resident_kernel<T, V, 256>), grid, dim3(256), lds, st, p);
        else
            hipLaunchKernelGGL((gn_bwd_resident_kernel<T, V, 512>), grid, dim3(512), lds, st, p);
        if (p.B > 1) hipLaunchKernelGGL(gn_bwd_affine_kernel, dim3(ceil_div(p.C, 64)), dim3(GN_T), 0, st, p);
        return;
    }
    p.chunks = stream_chunks(p.B, p.n);
    p.rows = ceil_div(p.n, p.chunks);
    hipLaunchKernelGGL((gn_bwd_sums_kernel<T, V>), dim3(p.chunks, p.B), dim3(GN_T), (size_t)GN_T * V * 8, st, p);
    hipLaunchKernelGGL(gn_bwd_reduce_kernel, dim3(ceil_div(p.C, 64), p.B), dim3(GN_T), 0, st, p);
    const size_t lds = (size_t)p.G * 8 > 4096 ? (size_t)p.G * 8 : 4096;
    hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V>), dim3(p.chunks, p.B + 1), dim3(GN_T), lds, st, p);
}

bool overlaps(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + nb && y < x + na;
}

// May `out` be written while `in` is read, both [rows, C] with their strides in bytes?  Yes if the ranges are apart, if
// it is the same matrix (every element is read before it is written, by the same thread), or if the two are column
// ranges of one wider matrix that share no column.
bool rows_ok(const void* in, size_t ldi, int ei, const void* out, size_t ldo, int eo, size_t rows, int C) {
    const size_t wi = (size_t)C * ei, wo = (size_t)C * eo, si = ldi * ei, so = ldo * eo;
    if (!overlaps(in, (rows - 1) * si + wi, out, (rows - 1) * so + wo)) return true;
    if (si != so) return false;
    if (in == out) return ei == eo;
    const uintptr_t x = (uintptr_t)in, y = (uintptr_t)out;
    const size_t d = y > x ? (y - x) % si : (si - (x - y) % si) % si;   // out's first column, seen from in's
    return d >= wi && d + wo <= si;
}

int check_common(const char* what, int B, int n, int C, int G, int act, size_t workspace_bytes) {
    UWIR_CHECK(B > 0 && B <= 65534 && n > 0 && C > 0 && C <= GN_MAX_C, "%s: bad shape (0 < B <= 65534, n > 0, 0 < C <= %d)", what,
               GN_MAX_C);
    UWIR_CHECK(G > 0 && C % G == 0, "%s: groups must divide C", what);
    UWIR_CHECK(act == UWIR_ACT_NONE || act == UWIR_ACT_SILU, "%s: act must be UWIR_ACT_NONE or UWIR_ACT_SILU", what);
    UWIR_CHECK(workspace_bytes >= uwir_group_norm_act_workspace_bytes(B, n, C, G), "%s: workspace too small", what);
    return UWIR_OK;
}

}  // namespace

// partials of the streamed form: per chunk and group (forward) or per chunk and channel (backward), and per image and channel
extern "C" size_t uwir_group_norm_act_workspace_bytes(int B, int n, int C, int groups) {
    if (B <= 0 || n <= 0 || C <= 0 || groups <= 0) return 0;
    const size_t ch = stream_chunks(B, n);
    const size_t fwd = (size_t)B * ch * groups * 16, bwd = al256((size_t)B * ch * C * 8) + (size_t)B * C * 8;
    return al256(fwd > bwd ? fwd : bwd);
}

extern "C" int uwir_group_norm_act(const void* x, int x_dtype, size_t ldx, int B, int n, int C, int groups, float eps,
                                   const float* gamma, const float* beta, const float* scale_shift, size_t ld_ss, int act,
                                   void* out, int out_dtype, size_t ldo, float* mean, float* rstd, void* workspace,
                                   size_t workspace_bytes, uwir_stream_t stream) {
    UWIR_CHECK(x && gamma && beta && out && workspace, "group_norm_act: null pointer");
    if (int rc = check_common("group_norm_act", B, n, C, groups, act, workspace_bytes)) return rc;
    UWIR_CHECK((x_dtype == UWIR_F32 || x_dtype == UWIR_BF16) && (out_dtype == UWIR_F32 || out_dtype == UWIR_BF16),
               "group_norm_act: bad dtype");
    UWIR_CHECK(ldx >= (size_t)C && ldo >= (size_t)C && (!scale_shift || ld_ss >= (size_t)2 * C),
               "group_norm_act: row strides must be at least C (2 C for scale_shift)");
    UWIR_CHECK(eps > 0.f, "group_norm_act: eps must be positive");
    UWIR_CHECK(((uintptr_t)workspace & 15) == 0, "group_norm_act: workspace must be 16-byte aligned");
    const int ex = x_dtype == UWIR_BF16 ? 2 : 4, eo = out_dtype == UWIR_BF16 ? 2 : 4;
    const size_t rows = (size_t)B * n, bx = ((rows - 1) * ldx + C) * ex, bo = ((rows - 1) * ldo + C) * eo;
    UWIR_CHECK(rows_ok(x, ldx, ex, out, ldo, eo, rows, C), "group_norm_act: x and out overlap");
    UWIR_CHECK(!overlaps(workspace, workspace_bytes, out, bo) && !overlaps(workspace, workspace_bytes, x, bx),
               "group_norm_act: the workspace overlaps x or out");
    GnArgs p = {};
    p.x = x; p.out = out; p.gamma = gamma; p.beta = beta; p.ss = scale_shift; p.mean = mean; p.rstd = rstd;
    p.part = (double2*)workspace;
    p.ldx = ldx; p.ldo = ldo; p.ld_ss = ld_ss;
    p.B = B; p.n = n; p.C = C; p.G = groups; p.cg = C / groups; p.eps = eps; p.act = act;
    // widest vector (16 bytes of x at most) that the channel count, strides and addresses allow
    int V = 16 / ex;
    while (V > 1 && (C % V || !vec_ok(x, ldx, V, ex) || !vec_ok(out, ldo, V, eo))) V >>= 1;
    hipStream_t st = (hipStream_t)stream;
    with_v(V, [&](auto v) {
        constexpr int W = decltype(v)::value;
        if (x_dtype == UWIR_BF16) {
            if (out_dtype == UWIR_BF16) launch_fwd<bf16_t, bf16_t, W>(p, st);
            else launch_fwd<bf16_t, float, W>(p, st);
        } else if constexpr (W <= 4) {
            if (out_dtype == UWIR_BF16) launch_fwd<float, bf16_t, W>(p, st);
            else launch_fwd<float, float, W>(p, st);
        }
        return 0;
    });
    UWIR_LAUNCH_CHECK("group_norm_act");
    return UWIR_OK;
}

extern "C" int uwir_group_norm_act_backward(const void* dy, size_t ldy, const void* x, size_t ldx, int dtype, int B, int n,
                                            int C, int groups, const float* gamma, const float* beta, const float* mean,
                                            const float* rstd, const float* scale_shift, size_t ld_ss, int act, void* dx,
                                            size_t ldd, float* dgamma, float* dbeta, float* dscale_shift, size_t ld_dss,
                                            void* workspace, size_t workspace_bytes, uwir_stream_t stream) {
    UWIR_CHECK(dy && x && gamma && beta && mean && rstd && dx && dgamma && dbeta && workspace,
               "group_norm_act_backward: null pointer");
    if (int rc = check_common("group_norm_act_backward", B, n, C, groups, act, workspace_bytes)) return rc;
    UWIR_CHECK(dtype == UWIR_F32 || dtype == UWIR_BF16, "group_norm_act_backward: bad dtype");
    UWIR_CHECK(ldx >= (size_t)C && ldy >= (size_t)C && ldd >= (size_t)C && (!scale_shift || ld_ss >= (size_t)2 * C) &&
                   (!dscale_shift || ld_dss >= (size_t)2 * C),
               "group_norm_act_backward: row strides must be at least C (2 C for scale_shift)");
    UWIR_CHECK(!dscale_shift || scale_shift, "group_norm_act_backward: dscale_shift without scale_shift");
    UWIR_CHECK(((uintptr_t)workspace & 15) == 0, "group_norm_act_backward: workspace must be 16-byte aligned");
    const int es = dtype == UWIR_BF16 ? 2 : 4;
    const size_t rows = (size_t)B * n, bx = ((rows - 1) * ldx + C) * es, by = ((rows - 1) * ldy + C) * es,
                 bo = ((rows - 1) * ldd + C) * es;
    UWIR_CHECK(rows_ok(x, ldx, es, dx, ldd, es, rows, C) && rows_ok(dy, ldy, es, dx, ldd, es, rows, C),
               "group_norm_act_backward: dx overlaps x or dy");
    UWIR_CHECK(!overlaps(workspace, workspace_bytes, dx, bo) && !overlaps(workspace, workspace_bytes, x, bx) &&
                   !overlaps(workspace, workspace_bytes, dy, by),
               "group_norm_act_backward: the workspace overlaps dy, x or dx");
    GnArgs p = {};
    p.x = x; p.dy = dy; p.out = dx; p.gamma = gamma; p.beta = beta; p.ss = scale_shift; p.mean_in = mean; p.rstd_in = rstd;
    p.dgamma = dgamma; p.dbeta = dbeta; p.dss = dscale_shift;
    p.ldx = ldx; p.ldy = ldy; p.ldo = ldd; p.ld_ss = ld_ss; p.ld_dss = ld_dss;
    p.B = B; p.n = n; p.C = C; p.G = groups; p.cg = C / groups; p.act = act;
    p.cpart = (float2*)workspace;
    p.csum = (float2*)((char*)workspace + al256((size_t)B * stream_chunks(B, n) * C * 8));
    int V = 16 / es;
    while (V > 1 && (C % V || !vec_ok(x, ldx, V, es) || !vec_ok(dy, ldy, V, es) || !vec_ok(dx, ldd, V, es))) V >>= 1;
    hipStream_t st = (hipStream_t)stream;
    with_v(V, [&](auto v) {
        constexpr int W = decltype(v)::value;
        if (dtype == UWIR_BF16) launch_bwd<bf16_t, W>(p, st);
        else if constexpr (W <= 4) launch_bwd<float, W>(p, st);
        return 0;
    });
    UWIR_LAUNCH_CHECK("group_norm_act_backward");
    return UWIR_OK;
}
