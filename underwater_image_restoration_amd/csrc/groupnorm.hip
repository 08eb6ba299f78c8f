// Group norm with an activation on NHWC rows, forward and backward.
//   mean, var over the n x cg elements of (image, group);  xh = (x - mean) rstd
//   z = (xh gamma + beta)(1 + scale_b) + shift_b;   y = act(z),  act = identity or SiLU
// Both directions are bound by memory (or, for small maps, by launch latency).  A block owns a slab of whole groups (at
// least 64 bytes of a row, 128 where the map is streamed: full cache lines) and some rows of one image:
//   resident  all rows: they stay in registers between the statistics and the output, every element is touched once and
//             there is one launch
//   streamed  a chunk of rows: statistics in one launch, output in the next; the second read of x comes from the L2 (the
//             same block index runs on the same XCD) or the memory-side cache where the map fits
// Statistics: every thread reduces batches of rows to (mean, sum of squared distances to that mean) per channel and
// merges them pairwise, so that a stray first element costs no digits and a mean far from zero costs the variance |mean| / sigma
// roundings, not the square of that; everything across
// threads is summed in fp64 in a fixed order (results do not depend on scheduling).
#include "common.h"
#include <type_traits>

namespace {

constexpr int GN_T = 512;          // threads of the streaming kernels
constexpr int GN_R = 8;            // rows a thread of the resident form holds
constexpr int GN_RS = 4;           // rows a thread of the streamed form loads ahead of using them
constexpr int GN_RUN = 128;        // rows that a thread of the streamed form adds up in fp32 before the sums move on to fp64
constexpr int GN_MAX_C = 2048;     // channels of a group, and so of a slab, are bounded by the per-slab sums in LDS
constexpr int GN_MAX_CHUNKS = 128; // row chunks of an image (each output block sums all partials of its slab)

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
    template <bool BYPASS = false> __device__ __forceinline__ void store(T* p) const {
        if constexpr (BYPASS) __builtin_nontemporal_store(v, reinterpret_cast<typename VecT<T, V>::type*>(p));
        else *reinterpret_cast<typename VecT<T, V>::type*>(p) = v;
    }
};

struct GnArgs {
    const void *x, *dy;
    void* out;                       // y, or dx
    const float *gamma, *beta, *ss;  // ss [B, ld_ss]: [scale | shift], or NULL
    const float *mean_in, *rstd_in;  // backward
    float *mean, *rstd;              // forward, optional
    float *dgamma, *dbeta, *dss;     // backward; dss [B, ld_dss] optional
    double2* part;                   // forward partials [B][G][chunks]: (sum, sum of squares)
    float2* cpart;                   // backward partials [B][chunks][C]: (sum dz, sum dz xh)
    float2* csum;                    // the same summed over the chunks, [B][C]
    const float2* sums;              // what the output pass reads: cpart or csum, [B][sum_chunks][C]
    size_t ldx, ldy, ldo, ld_ss, ld_dss;
    double inv_n;                    // 1 / (n cg)
    int B, n, C, G, cg, chunks, rows, slab, sum_chunks;  // rows per chunk; channels per slab
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
    // merge `k` <= R fresh rows (pairwise update: exact in the count weights)
    template <int R, bool FULL, typename T> __device__ __forceinline__ void merge(const Pack<T, V>* p, int k) {
        const float inv = FULL ? 1.f / R : 1.f / (float)k;
        const float wa = (float)k * __builtin_amdgcn_rcpf((float)(cnt + k)), wb = (float)cnt * wa;   // weights: an ulp is harmless
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < R; ++i) s += FULL || i < k ? p[i].get(j) : 0.f;
            const float m = s * inv;
            float q = 0.f;
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const float d = FULL || i < k ? p[i].get(j) - m : 0.f;
                q = fmaf(d, d, q);
            }
            const float d = m - mean[j];
            mean[j] = fmaf(d, wa, mean[j]);
            m2[j] += fmaf(d, d * wb, q);   // of the first batch d is the mean itself, whose square may leave the range, and wb 0
        }
        cnt += k;
    }
    template <int R, typename T> __device__ __forceinline__ void batch(const Pack<T, V>* p, int k) {
        if (k == R) merge<R, true>(p, k);
        else if (k > 0) merge<R, false>(p, k);
    }
    // channels of one group put together, `u` neighbours at a time (a power of two): V / u entries remain in front
    __device__ __forceinline__ void fold(int u) {
        float half = 0.5f * (float)cnt;
#pragma unroll
        for (int w = V; w > 1; w >>= 1)
            if (u * w > V) {   // another halving
#pragma unroll
                for (int j = 0; j < w / 2; ++j) {
                    const float d = mean[2 * j] - mean[2 * j + 1];
                    m2[j] = m2[2 * j] + m2[2 * j + 1] + half * d * d;
                    mean[j] = 0.5f * (mean[2 * j] + mean[2 * j + 1]);
                }
                half *= 2.f;
            }
    }
};

// neighbouring channels of a thread that always lie in one group
template <int V> __device__ __forceinline__ int fold_of(int cg) {
    return cg % V == 0 ? V : (V % cg == 0 ? cg : 1);
}

// rows r, r + step, ... (k <= R of them; the others repeat row r, which must exist)
template <int R, typename T, int V>
__device__ __forceinline__ void load_rows(Pack<T, V>* buf, const T* src, size_t ld, int r, int step, int k) {
#pragma unroll
    for (int i = 0; i < R; ++i) buf[i].load(src + (size_t)(i < k ? r + i * step : r) * ld);
}

// walks a thread's rows r, r + step, ... < r1: f(r, R) for full batches of R rows (k is then a constant), f(r, k) for the rest
template <int R, typename F> __device__ __forceinline__ void row_batches(int r, int r1, int step, F f) {
    for (; r + (R - 1) * step < r1; r += R * step) f(r, R);
    if (r < r1) f(r, (r1 - r + step - 1) / step);
}

__device__ __forceinline__ double shfl_xor_d(double v, int m) {
    return __hiloint2double(__shfl_xor(__double2hiint(v), m), __shfl_xor(__double2loint(v), m));
}

// For every group g of a block: add(g, lane, lanes, s, q) sums the share of one of `lanes` lanes, done(g, s, q) gets the total
// in one thread.  Teams of up to a wave; with fewer groups than teams several teams share a group and `scratch` [T / 64] joins
// them.  Ends with a barrier.
template <int T, typename F, typename D>
__device__ __forceinline__ void group_sums(int G, int tid, double2* scratch, F add, D done) {
    int tpg = 64;
    while (tpg > 1 && tpg * G > T) tpg >>= 1;
    const int teams = T / tpg, lane = tid & (tpg - 1), team = tid / tpg;
    if (G * 2 <= teams) {   // only with whole-wave teams
        const int parts = teams / G, g = team % G, part = team / G;
        double a = 0., b = 0.;
        if (part < parts) add(g, part * 64 + lane, parts * 64, a, b);
        for (int o = 32; o; o >>= 1) {
            a += shfl_xor_d(a, o);
            b += shfl_xor_d(b, o);
        }
        if (lane == 0) scratch[team] = make_double2(a, b);
        __syncthreads();
        if (tid < G) {
            a = b = 0.;
            for (int q = 0; q < parts; ++q) {
                a += scratch[q * G + tid].x;
                b += scratch[q * G + tid].y;
            }
            done(tid, a, b);
        }
    } else {
        for (int g0 = 0; g0 < G; g0 += teams) {   // uniform trip count: the shuffles see whole waves
            const int g = g0 + team;
            double a = 0., b = 0.;
            if (g < G) add(g, lane, tpg, a, b);
            for (int o = tpg >> 1; o; o >>= 1) {
                a += shfl_xor_d(a, o);
                b += shfl_xor_d(b, o);
            }
            if (g < G && lane == 0) done(g, a, b);
        }
    }
    __syncthreads();
}

// the same over m items a group, item i from f(g, i)
template <int T, typename F, typename D>
__device__ __forceinline__ void group_items(int G, int m, int tid, double2* scratch, F f, D done) {
    group_sums<T>(G, tid, scratch,
                  [&](int g, int lane, int lanes, double& s, double& q) {
                      for (int i = lane; i < m; i += lanes) {
                          const double2 v = f(g, i);
                          s += v.x;
                          q += v.y;
                      }
                  },
                  done);
}

__device__ __forceinline__ float act_silu(float z) { return z * sigmoid_fast(z); }
__device__ __forceinline__ float dact_silu(float z) {
    const float s = sigmoid_fast(z);
    return s * fmaf(z, 1.f - s, 1.f);
}

// where a block's thread works: its slab of one image, a vector of V channels, row lane rl of RL
struct Place {
    int b, ch0, sc, tw, RL, cv, rl;
    template <int V> __device__ __forceinline__ static Place of(const GnArgs& p, int slab, int b, int tid, int T) {
        Place l;
        l.b = b;
        l.ch0 = slab * p.slab;
        l.sc = min(p.slab, p.C - l.ch0);
        l.tw = l.sc / V;
        // quotients of numbers below 2^11 through the reciprocal: (a + 1/2) / b is at least 1 / (2 b) away from an integer
        const float inv = __builtin_amdgcn_rcpf((float)l.tw);
        l.RL = l.tw <= T ? (int)((T + 0.5f) * inv) : 1;
        l.rl = (int)((tid + 0.5f) * inv);
        l.cv = tid - l.rl * l.tw;
        return l;
    }
};

// a thread's folded statistics -> LDS, V / fold entries a thread
template <int V> __device__ __forceinline__ void put_stats(Stat<V>& st, int fold, int tid, float* sm, float* sq) {
    st.fold(fold);
    const int e = V / fold;
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (j < e) {
            sm[tid * e + j] = st.mean[j];
            sq[tid * e + j] = st.m2[j];
        }
    __syncthreads();
}

// Sums of the block's rows per group from the threads' statistics in LDS: `fold` channels an entry, `total` rows dealt to RL
// row lanes in turn.  A lane of a group's team keeps to one entry column, or (more columns than lanes) to whole columns.
template <int T, int V, typename D>
__device__ __forceinline__ void slab_group_sums(const GnArgs& p, const Place& l, int fold, int total, const float* sm, const float* sq,
                                                double2* scratch, int tid, D done) {
    const int rows = min(l.RL, max(total, 0)), base = total > 0 ? total / l.RL : 0, rem = total > 0 ? total % l.RL : 0;
    const int width = l.sc / fold, ce = p.cg / fold, groups = l.sc / p.cg;
    group_sums<T>(groups, tid, scratch,
                  [&](int g, int lane, int lanes, double& s, double& q) {
                      const int rl = ce < lanes ? lanes / ce : 1, r0 = ce < lanes ? lane / ce : 0;
                      if (r0 >= rl) return;
                      for (int c = ce < lanes ? lane - r0 * ce : lane; c < ce; c += ce < lanes ? ce : lanes)
                          for (int r = r0; r < rows; r += rl) {
                              const int at = r * width + g * ce + c;
                              const double k = (double)((base + (r < rem)) * fold), m = sm[at];
                              s += k * m;
                              q += (double)sq[at] + k * m * m;
                          }
                  },
                  done);
}

__device__ __forceinline__ float2 finish_stats(double s, double q, double inv_n, float eps) {
    const double m = s * inv_n;
    const float v = (float)(q * inv_n - m * m);
    return make_float2((float)m, rsqrtf((v < 0.f ? 0.f : v) + eps));   // (a NaN stays one)
}

// V consecutive floats at any alignment of 4 bytes, 16 bytes at a time
template <int V> __device__ __forceinline__ void load_floats(const float* p, float* o) {
    if constexpr (V % 4 == 0) {
#pragma unroll
        for (int j = 0; j < V; j += 4) __builtin_memcpy(o + j, p + j, 16);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = p[j];
    }
}

// f(j, g) for the channels c0 + j, j < V, of a slab and the group g each lies in
template <int V, typename F> __device__ __forceinline__ void each_group(int c0, int cg, F f) {
    int g = c0 / cg, at = c0 - g * cg;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        f(j, g);
        if (++at == cg) at = 0, ++g;
    }
}

// per-channel coefficients of a thread's V channels: z = (x - m) a + s, xh = (x - m) r; gamma, beta and the modulation are
// loaded ahead of the statistics
template <int V> struct Coef {
    float w[V], s[V], m[V], r[V];   // w = gamma (1 + scale)
    __device__ __forceinline__ void load(const GnArgs& p, int b, int c0) {
        load_floats<V>(p.gamma + c0, w);
        load_floats<V>(p.beta + c0, s);
        if (p.ss) {
            float f[V], h[V];
            load_floats<V>(p.ss + (size_t)b * p.ld_ss + c0, f);
            load_floats<V>(p.ss + (size_t)b * p.ld_ss + p.C + c0, h);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                w[j] *= 1.f + f[j];
                s[j] = fmaf(s[j], 1.f + f[j], h[j]);
            }
        }
    }
    __device__ __forceinline__ void stats(int j, float mean, float rstd) {
        m[j] = mean;
        r[j] = rstd;
        w[j] *= rstd;               // now a
    }
    __device__ __forceinline__ float z(int j, float d) const { return fmaf(d, w[j], s[j]); }
};

template <int R, bool BYPASS = false, typename TX, typename TO, int V>
__device__ __forceinline__ void emit(const Pack<TX, V>* buf, const Coef<V>& co, TO* dst, size_t ld, int r, int step, int k, bool silu) {
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (i < k) {
            Pack<TO, V> o;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float z = co.z(j, buf[i].get(j) - co.m[j]);
                o.set(j, silu ? act_silu(z) : z);
            }
            o.template store<BYPASS>(dst + (size_t)(r + i * step) * ld);
        }
}

// ---------------------------------------------------------------------------------------- forward, streamed
// Bound by reading x once: 16 x 256 x 256 x 64 bf16 (134 MB) in 22.2 us, 6.0 TB/s, 8 x 64 x 64 x 256 (17 MB) in 5.8 us.  A chunk of
// rows per block, one block per CU: 3 us of every block are its start, the reductions across threads and its end.
// A slab wider than the block (one group over more than GN_T vectors) is walked in tiles of GN_T vectors; the groups are then
// summed tile by tile through `ch`.
template <typename TX, int V>
__global__ void __launch_bounds__(GN_T) gn_stats_kernel(GnArgs p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    double2* scratch = reinterpret_cast<double2*>(smem);               // [GN_T / 64]
    float* sm = reinterpret_cast<float*>(scratch + GN_T / 64);         // [GN_T][V] means
    float* sq = sm + GN_T * V;                                         // [GN_T][V] squares
    const int tid = threadIdx.x, chunk = blockIdx.x, b = blockIdx.z;
    const Place l = Place::of<V>(p, blockIdx.y, b, tid, GN_T);
    const int r0 = chunk * p.rows, r1 = min(p.n, r0 + p.rows);
    const TX* X = (const TX*)p.x + (size_t)b * p.n * p.ldx + l.ch0;
    double2* out = p.part + ((size_t)b * p.G + l.ch0 / p.cg) * p.chunks + chunk;
    double wide_s = 0., wide_q = 0.;
    for (int v0 = 0; v0 < l.tw; v0 += GN_T) {
        const bool wide = l.tw > GN_T;
        const int cv = wide ? v0 + tid : l.cv;
        const TX* src = X + (size_t)cv * V;
        int g0 = r0;
        do {   // runs of GN_RUN rows a thread (one but for many large images; none where a chunk is empty)
            const int g1 = min(r1, g0 + l.RL * GN_RUN);
            Stat<V> st;
            st.clear();
            if (wide ? cv < l.tw : l.rl < l.RL)
                row_batches<GN_RS>(g0 + (wide ? 0 : l.rl), g1, l.RL, [&](int r, int k) {
                    Pack<TX, V> buf[GN_RS];
                    load_rows<GN_RS>(buf, src, p.ldx, r, l.RL, k);
                    st.template batch<GN_RS>(buf, k);
                });
            if (wide) {   // a single group: the thread's own sums
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const double k = st.cnt, m = st.mean[j];
                    wide_s += k * m;
                    wide_q += (double)st.m2[j] + k * m * m;
                }
                continue;
            }
            const int fold = fold_of<V>(p.cg);
            put_stats(st, fold, tid, sm, sq);
            slab_group_sums<GN_T, V>(p, l, fold, g1 - g0, sm, sq, scratch, tid, [&](int g, double s, double q) {
                double2& o = out[(size_t)g * p.chunks];   // the same thread's every time
                o = g0 == r0 ? make_double2(s, q) : make_double2(o.x + s, o.y + q);
            });
        } while ((g0 += l.RL * GN_RUN) < r1);
    }
    if (l.tw > GN_T) {
        double2* all = scratch + GN_T / 64;   // [GN_T], in the place of sm and sq
        all[tid] = make_double2(wide_s, wide_q);
        __syncthreads();
        group_items<GN_T>(1, GN_T, tid, scratch, [&](int, int i) { return all[i]; },
                         [&](int, double s, double q) { out[0] = make_double2(s, q); });
    }
}

// y = act(a x + s) with a = rstd gamma (1 + scale), s = (beta - mean rstd gamma)(1 + scale) + shift held per thread for its V
// channels.  Bound by bytes: x again (from the memory-side cache) and y out; the first rows are loaded before the partials are
// summed.  16 x 256 x 256 x 64 bf16 43.8 us (268 MB, 6.1 TB/s), 8 x 64 x 64 x 256 9.3 us (34 MB; the partials' sums take 3 of them).
template <typename TX, typename TO, int V, bool BYPASS>
__global__ void __launch_bounds__(GN_T, 4) gn_apply_kernel(GnArgs p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    double2* scratch = reinterpret_cast<double2*>(smem);               // [GN_T / 64]
    float2* gst = reinterpret_cast<float2*>(scratch + GN_T / 64);      // [slab / cg] (mean, rstd)
    const int tid = threadIdx.x, chunk = blockIdx.x, b = blockIdx.z;
    const Place l = Place::of<V>(p, blockIdx.y, b, tid, GN_T);
    const int cg = p.cg, g0 = l.ch0 / cg;
    const int r0 = chunk * p.rows, r1 = min(p.n, r0 + p.rows);
    const TX* X = (const TX*)p.x + (size_t)b * p.n * p.ldx + l.ch0;
    TO* Y = (TO*)p.out + (size_t)b * p.n * p.ldo + l.ch0;
    const bool silu = p.act == UWIR_ACT_SILU, wide = l.tw > GN_T;
    // the first rows and the coefficients are on their way while the statistics are put together
    Coef<V> co;
    Pack<TX, V> buf[GN_RS];
    const int ra = r0 + l.rl, rest = wide || l.rl >= l.RL || ra >= r1 ? 0 : (r1 - ra + l.RL - 1) / l.RL, ka = min(rest, GN_RS);
    if (rest) {
        load_rows<GN_RS>(buf, X + l.cv * V, p.ldx, ra, l.RL, ka);
        co.load(p, b, l.ch0 + l.cv * V);
    }
    const double2* part = p.part + ((size_t)b * p.G + g0) * p.chunks;
    group_items<GN_T>(l.sc / cg, p.chunks, tid, scratch, [&](int g, int i) { return part[(size_t)g * p.chunks + i]; },
                     [&](int g, double s, double q) {
                         const float2 st = finish_stats(s, q, p.inv_n, p.eps);
                         gst[g] = st;
                         if (chunk == 0) {
                             if (p.mean) p.mean[(size_t)b * p.G + g0 + g] = st.x;
                             if (p.rstd) p.rstd[(size_t)b * p.G + g0 + g] = st.y;
                         }
                     });
    auto finish = [&](int cv) { each_group<V>(cv * V, cg, [&](int j, int g) { co.stats(j, gst[g].x, gst[g].y); }); };
    auto walk = [&](int cv, int r, int step) {
        row_batches<GN_RS>(r, r1, step, [&](int r, int k) {
            load_rows<GN_RS>(buf, X + cv * V, p.ldx, r, step, k);
            emit<GN_RS, BYPASS>(buf, co, Y + cv * V, p.ldo, r, step, k, silu);
        });
    };
    if (rest) {
        finish(l.cv);
        emit<GN_RS, BYPASS>(buf, co, Y + l.cv * V, p.ldo, ra, l.RL, ka, silu);
        walk(l.cv, ra + GN_RS * l.RL, l.RL);
    }
    if (wide)
        for (int cv = tid; cv < l.tw; cv += GN_T) {
            co.load(p, b, l.ch0 + cv * V);
            finish(cv);
            walk(cv, r0, 1);
        }
}

// ---------------------------------------------------------------------------------------- forward, resident
// All rows of a slab in a block's registers (GN_R a thread).  Bound by latency: a launch, one load, two sums across the block, one
// store; 1 x 8 x 8 x 512 fp32 5.1 us, of which an empty kernel takes 2.
template <typename TX, typename TO, int V, int T>
__global__ void __launch_bounds__(T) gn_resident_kernel(GnArgs p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float* sm = reinterpret_cast<float*>(smem);
    float* sq = sm + T * V;
    double2* scratch = reinterpret_cast<double2*>(sq + T * V);         // [T / 64]
    float2* gst = reinterpret_cast<float2*>(scratch + T / 64);         // [slab / cg]
    const int tid = threadIdx.x, b = blockIdx.y, cg = p.cg;
    const Place l = Place::of<V>(p, blockIdx.x, b, tid, T);
    const int g0 = l.ch0 / cg;
    const TX* X = (const TX*)p.x + (size_t)b * p.n * p.ldx + l.ch0 + l.cv * V;
    Pack<TX, V> buf[GN_R];
    Coef<V> co;
    const int k = l.rl < l.RL && l.rl < p.n ? (p.n - l.rl + l.RL - 1) / l.RL : 0;  // <= GN_R by the launch rule
    if (k > 0) {
        load_rows<GN_R>(buf, X, p.ldx, l.rl, l.RL, k);
        co.load(p, b, l.ch0 + l.cv * V);
    }
    Stat<V> st;
    st.clear();
    st.template batch<GN_R>(buf, k);
    const int fold = fold_of<V>(cg);
    put_stats(st, fold, tid, sm, sq);
    slab_group_sums<T, V>(p, l, fold, p.n, sm, sq, scratch, tid, [&](int g, double s, double q) {
        const float2 f = finish_stats(s, q, p.inv_n, p.eps);
        gst[g] = f;
        if (p.mean) p.mean[(size_t)b * p.G + g0 + g] = f.x;
        if (p.rstd) p.rstd[(size_t)b * p.G + g0 + g] = f.y;
    });
    if (k <= 0) return;
    each_group<V>(l.cv * V, cg, [&](int j, int g) { co.stats(j, gst[g].x, gst[g].y); });
    emit<GN_R>(buf, co, (TO*)p.out + (size_t)b * p.n * p.ldo + l.ch0 + l.cv * V, p.ldo, l.rl, l.RL, k, p.act == UWIR_ACT_SILU);
}

// ---------------------------------------------------------------------------------------- backward
// SiLU's derivative costs an exponential and a reciprocal per element (8 of about 20 issue slots): in the bf16 passes vector work
// takes half to two thirds of the cycles (counted), little of it under the loads with two waves a SIMD.  With d = x - m the sums need dz and dz d only (xh = d r enters once per channel).
template <int V, typename T>
__device__ __forceinline__ void bwd_stats(const GnArgs& p, Coef<V>& co, int b, int c0) {
    co.load(p, b, c0);
    const float *m = p.mean_in + (size_t)b * p.G, *r = p.rstd_in + (size_t)b * p.G;
    each_group<V>(c0, p.cg, [&](int j, int g) { co.stats(j, m[g], r[g]); });
}

// adds a batch of rows: s1 += sum dz, s2 += sum dz d, each summed within the batch first
template <int R, typename T, int V>
__device__ __forceinline__ void bwd_batch(const Pack<T, V>* bx, const Pack<T, V>* bd, const Coef<V>& co, int k, bool silu, float* s1,
                                          float* s2) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
        float t1 = 0.f, t2 = 0.f;
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (i < k) {
                const float d = bx[i].get(j) - co.m[j];
                float dz = bd[i].get(j);
                if (silu) dz *= dact_silu(co.z(j, d));
                t1 += dz;
                t2 = fmaf(dz, d, t2);
            }
        s1[j] += t1;
        s2[j] += t2;
    }
}

// dx = r (w dz - m1 - xh m2) with u1 = r m1, u2 = r^2 m2
template <int R, bool BYPASS = false, typename T, int V>
__device__ __forceinline__ void bwd_emit(const Pack<T, V>* bx, const Pack<T, V>* bd, const Coef<V>& co, const float* u1, const float* u2,
                                         T* dst, size_t ld, int r, int step, int k, bool silu) {
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (i < k) {
            Pack<T, V> o;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = bx[i].get(j) - co.m[j];
                float dz = bd[i].get(j);
                if (silu) dz *= dact_silu(co.z(j, d));
                o.set(j, fmaf(co.w[j], dz, -fmaf(d, u2[j], u1[j])));
            }
            o.template store<BYPASS>(dst + (size_t)(r + i * step) * ld);
        }
}

// S1 = sum dz, S2 = sum dz xh per channel over a chunk of rows, dz = dy act'(z).  Bound by reading x and dy and, with SiLU, by the
// exponential and reciprocal per element: 8 x 128 x 128 x 128 bf16 16.3 us (67 MB, 4.1 TB/s), 8 x 256 x 256 x 64 fp32 38.8 us
// (268 MB, 6.9 TB/s).
constexpr int GN_RB = 2;   // rows a thread has in flight, x and dy each: coefficients fill the registers, waves hide the latency

template <typename T, int V>
__global__ void __launch_bounds__(GN_T, 4) gn_bwd_sums_kernel(GnArgs p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float2* red = reinterpret_cast<float2*>(smem);             // [GN_T][V]
    double2* run = reinterpret_cast<double2*>(red + GN_T * V); // [slab]
    const int tid = threadIdx.x, chunk = blockIdx.x, b = blockIdx.z;
    const Place l = Place::of<V>(p, blockIdx.y, b, tid, GN_T);
    const int r0 = chunk * p.rows, r1 = min(p.n, r0 + p.rows);
    const T* X = (const T*)p.x + (size_t)b * p.n * p.ldx + l.ch0;
    const T* DY = (const T*)p.dy + (size_t)b * p.n * p.ldy + l.ch0;
    float2* out = p.cpart + ((size_t)b * p.chunks + chunk) * p.C + l.ch0;
    const bool silu = p.act == UWIR_ACT_SILU;
    for (int v0 = 0; v0 < l.tw; v0 += GN_T) {
        const bool wide = l.tw > GN_T;
        const int cv = wide ? v0 + tid : l.cv;
        const bool mine = wide ? cv < l.tw : l.rl < l.RL;
        Coef<V> co;
        if (mine) bwd_stats<V, T>(p, co, b, l.ch0 + cv * V);
        int g0 = r0;
        bool more;
        do {   // runs of GN_RUN rows a thread (one but for many large images; none where a chunk is empty)
            const int g1 = min(r1, g0 + l.RL * GN_RUN);
            more = g0 + l.RL * GN_RUN < r1;
            // a channel's sums: to memory after the last run, into `run` (by the same thread every time) before
            auto put = [&](int c, double a, double q) {
                if (g0 != r0) {
                    a += run[c].x;
                    q += run[c].y;
                }
                if (more) run[c] = make_double2(a, q);
                else out[c] = make_float2((float)a, (float)q);
            };
            float s1[V], s2[V];
#pragma unroll
            for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.f;
            if (mine) {
                row_batches<GN_RB>(g0 + (wide ? 0 : l.rl), g1, l.RL, [&](int r, int k) {
                    Pack<T, V> bx[GN_RB], bd[GN_RB];
                    load_rows<GN_RB>(bx, X + cv * V, p.ldx, r, l.RL, k);
                    load_rows<GN_RB>(bd, DY + cv * V, p.ldy, r, l.RL, k);
                    bwd_batch<GN_RB>(bx, bd, co, k, silu, s1, s2);
                });
#pragma unroll
                for (int j = 0; j < V; ++j) s2[j] *= co.r[j];
            }
            if (wide) {
                if (mine)
#pragma unroll
                    for (int j = 0; j < V; ++j) put(cv * V + j, s1[j], s2[j]);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) red[tid * V + j] = make_float2(s1[j], s2[j]);
                __syncthreads();
                // a team of T / width threads per channel (a power of two within a wave) over the row lanes
                int team = 1;
                while (team < 64 && team * 2 * l.sc <= GN_T) team *= 2;
                for (int c0 = 0; c0 < l.sc; c0 += GN_T / team) {
                    const int c = c0 + tid / team;
                    double a = 0., q = 0.;
                    if (c < l.sc)
                        for (int i = tid & (team - 1); i < l.RL; i += team) {
                            const float2 v = red[i * l.sc + c];
                            a += v.x;
                            q += v.y;
                        }
                    for (int o = team >> 1; o; o >>= 1) {
                        a += shfl_xor_d(a, o);
                        q += shfl_xor_d(q, o);
                    }
                    if (c < l.sc && (tid & (team - 1)) == 0) put(c, a, q);
                }
                if (more) __syncthreads();
            }
            g0 += l.RL * GN_RUN;
        } while (more);
    }
}

// sums over the chunks of 64 channels of one image, 8 lanes a channel: ahead of the output pass where a slab's partials are
// too many for every output block to read
__global__ void __launch_bounds__(GN_T) gn_bwd_reduce_kernel(GnArgs p) {
    __shared__ double2 red[8][64];
    const int cl = threadIdx.x & 63, l = threadIdx.x >> 6, c = blockIdx.x * 64 + cl, b = blockIdx.y;
    double a = 0., q = 0.;
    if (c < p.C)
        for (int i = l; i < p.chunks; i += 8) {
            const float2 v = p.cpart[((size_t)b * p.chunks + i) * p.C + c];
            a += v.x;
            q += v.y;
        }
    red[l][cl] = make_double2(a, q);
    __syncthreads();
    if (l == 0 && c < p.C) {
        for (int i = 1; i < 8; ++i) {
            a += red[i][cl].x;
            q += red[i][cl].y;
        }
        p.csum[(size_t)b * p.C + c] = make_float2((float)a, (float)q);
    }
}

// dgamma, dbeta of 64 channels: 8 lanes a channel over the images (and their chunks)
__device__ __forceinline__ void affine_grads(const GnArgs& p, int tile, double2 (*red)[64]) {
    const int cl = threadIdx.x & 63, l = threadIdx.x >> 6, c = tile * 64 + cl;
    double dg = 0., db = 0.;
    if (c < p.C)
        for (int b = l; b < p.B; b += 8) {
            const double f = p.ss ? 1. + (double)p.ss[(size_t)b * p.ld_ss + c] : 1.;
            for (int i = 0; i < p.sum_chunks; ++i) {
                const float2 v = p.sums[((size_t)b * p.sum_chunks + i) * p.C + c];
                dg += f * v.y;
                db += f * v.x;
            }
        }
    red[l][cl] = make_double2(dg, db);
    __syncthreads();
    if (l == 0 && c < p.C) {
        for (int i = 1; i < 8; ++i) {
            dg += red[i][cl].x;
            db += red[i][cl].y;
        }
        p.dgamma[c] = (float)dg;
        p.dbeta[c] = (float)db;
    }
}

// dgamma, dbeta (summed over the images in order) and dscale, dshift from the per-image sums: C B values, latency only (2 us)
__global__ void __launch_bounds__(GN_T) gn_bwd_affine_kernel(GnArgs p) {
    __shared__ double2 red[8][64];
    affine_grads(p, blockIdx.x, red);
}

// the modulation's gradient of one channel
__device__ __forceinline__ void put_dss(const GnArgs& p, int b, int c, double s1, double s2) {
    if (!p.dss) return;
    p.dss[(size_t)b * p.ld_dss + c] = (float)(p.gamma[c] * s2 + p.beta[c] * s1);
    p.dss[(size_t)b * p.ld_dss + p.C + c] = (float)s1;
}

// dx = rstd (w dz - m1 - xh m2), w = gamma (1 + scale), m1 and m2 the group's means of w S1 and w S2.  Bound like the sums' pass, with
// dx to write: 21.8 us (4.6 TB/s, both reads from the memory-side cache) and 63 us (403 MB, 6.4 TB/s) at the same two sizes.
// output pass; the last row of blocks (b == B) forms dgamma, dbeta instead
template <typename T, int V, bool BYPASS>
__global__ void __launch_bounds__(GN_T, 4) gn_bwd_apply_kernel(GnArgs p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, chunk = blockIdx.x, b = blockIdx.z;
    if (b == p.B) {
        for (int t = chunk + blockIdx.y * gridDim.x; t * 64 < p.C; t += gridDim.x * gridDim.y) {
            affine_grads(p, t, reinterpret_cast<double2(*)[64]>(smem));
            __syncthreads();
        }
        return;
    }
    double2* scratch = reinterpret_cast<double2*>(smem);            // [GN_T / 64]
    double2* ch = scratch + GN_T / 64;                              // [max(slab, GN_T)] sums, then w (S1, S2)
    float2* gm = reinterpret_cast<float2*>(ch + max(p.slab, GN_T)); // [slab / cg] (m1, m2)
    const Place l = Place::of<V>(p, blockIdx.y, b, tid, GN_T);
    const int cg = p.cg;
    const int r0 = chunk * p.rows, r1 = min(p.n, r0 + p.rows);
    const T* X = (const T*)p.x + (size_t)b * p.n * p.ldx + l.ch0;
    const T* DY = (const T*)p.dy + (size_t)b * p.n * p.ldy + l.ch0;
    T* DX = (T*)p.out + (size_t)b * p.n * p.ldo + l.ch0;
    const bool silu = p.act == UWIR_ACT_SILU, wide = l.tw > GN_T;
    // the first rows and the coefficients are on their way while the sums are put together
    Coef<V> co;
    Pack<T, V> bx[GN_RB], bd[GN_RB];
    const int ra = r0 + l.rl, rest = wide || l.rl >= l.RL || ra >= r1 ? 0 : (r1 - ra + l.RL - 1) / l.RL, ka = min(rest, GN_RB);
    if (rest) {
        load_rows<GN_RB>(bx, X + l.cv * V, p.ldx, ra, l.RL, ka);
        load_rows<GN_RB>(bd, DY + l.cv * V, p.ldy, ra, l.RL, ka);
        bwd_stats<V, T>(p, co, b, l.ch0 + l.cv * V);
    }
    // the slab's channel sums: lanes of a channel share the chunks, and are joined in LDS (a wide slab has one lane each)
    const int lanes = l.sc < GN_T ? GN_T / l.sc : 1, cl = l.sc < GN_T ? tid % l.sc : tid, ln = l.sc < GN_T ? tid / l.sc : 0;
    for (int c = cl; c < l.sc && ln < lanes; c += GN_T) {
        double a = 0., q = 0.;
        const float2* src = p.sums + (size_t)b * p.sum_chunks * p.C + l.ch0 + c;
#pragma unroll 4
        for (int i = ln; i < p.sum_chunks; i += lanes) {
            const float2 v = src[(size_t)i * p.C];
            a += v.x;
            q += v.y;
        }
        ch[ln * l.sc + c] = make_double2(a, q);
    }
    __syncthreads();
    for (int c = tid; c < l.sc; c += GN_T) {
        double2 v = ch[c];
        for (int i = 1; i < lanes; ++i) {
            v.x += ch[i * l.sc + c].x;
            v.y += ch[i * l.sc + c].y;
        }
        const int cc = l.ch0 + c;
        const double w = (double)p.gamma[cc] * (p.ss ? 1. + (double)p.ss[(size_t)b * p.ld_ss + cc] : 1.);
        if (chunk == 0) put_dss(p, b, cc, v.x, v.y);
        ch[c] = make_double2(w * v.x, w * v.y);
    }
    __syncthreads();
    group_items<GN_T>(l.sc / cg, cg, tid, scratch, [&](int g, int i) { return ch[g * cg + i]; },
                     [&](int g, double s, double q) { gm[g] = make_float2((float)(s * p.inv_n), (float)(q * p.inv_n)); });
    float u1[V], u2[V];
    auto finish = [&](int cv) {
        each_group<V>(cv * V, cg, [&](int j, int g) {
            u1[j] = co.r[j] * gm[g].x;
            u2[j] = co.r[j] * co.r[j] * gm[g].y;
        });
    };
    auto walk = [&](int cv, int r, int step) {
        row_batches<GN_RB>(r, r1, step, [&](int r, int k) {
            load_rows<GN_RB>(bx, X + cv * V, p.ldx, r, step, k);
            load_rows<GN_RB>(bd, DY + cv * V, p.ldy, r, step, k);
            bwd_emit<GN_RB, BYPASS>(bx, bd, co, u1, u2, DX + cv * V, p.ldo, r, step, k, silu);
        });
    };
    if (rest) {
        finish(l.cv);
        bwd_emit<GN_RB, BYPASS>(bx, bd, co, u1, u2, DX + l.cv * V, p.ldo, ra, l.RL, ka, silu);
        walk(l.cv, ra + GN_RB * l.RL, l.RL);
    }
    if (wide)
        for (int cv = tid; cv < l.tw; cv += GN_T) {
            bwd_stats<V, T>(p, co, b, l.ch0 + cv * V);
            finish(cv);
            walk(cv, r0, 1);
        }
}

// All rows of a slab in a block's registers, x and dy read once; per-channel sums leave for gn_bwd_affine_kernel's launch.  Bound by
// latency: 3 x 19 x 22 x 96 fp32 7.6 us and 2.0 us.
template <typename T, int V, int TH>
__global__ void __launch_bounds__(TH) gn_bwd_resident_kernel(GnArgs p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float2* red = reinterpret_cast<float2*>(smem);                     // [TH][V]
    double2* scratch = reinterpret_cast<double2*>(red + TH * V);       // [TH / 64]
    double2* ch = scratch + TH / 64;                                   // [slab] w (S1, S2)
    float2* gm = reinterpret_cast<float2*>(ch + p.slab);               // [slab / cg]
    const int tid = threadIdx.x, b = blockIdx.y, cg = p.cg;
    const Place l = Place::of<V>(p, blockIdx.x, b, tid, TH);
    const int cb = l.ch0 + l.cv * V;
    const T* X = (const T*)p.x + (size_t)b * p.n * p.ldx + cb;
    const T* DY = (const T*)p.dy + (size_t)b * p.n * p.ldy + cb;
    const bool silu = p.act == UWIR_ACT_SILU;
    const int k = l.rl < l.RL && l.rl < p.n ? (p.n - l.rl + l.RL - 1) / l.RL : 0;
    Pack<T, V> bx[GN_R], bd[GN_R];
    Coef<V> co;
    float s1[V], s2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.f;
    if (k > 0) {
        load_rows<GN_R>(bx, X, p.ldx, l.rl, l.RL, k);
        load_rows<GN_R>(bd, DY, p.ldy, l.rl, l.RL, k);
        bwd_stats<V, T>(p, co, b, cb);
        bwd_batch<GN_R>(bx, bd, co, k, silu, s1, s2);
#pragma unroll
        for (int j = 0; j < V; ++j) s2[j] *= co.r[j];
    }
#pragma unroll
    for (int j = 0; j < V; ++j) red[tid * V + j] = make_float2(s1[j], s2[j]);
    __syncthreads();
    const int rows = min(l.RL, p.n);
    int team = 1;
    while (team < 64 && team * 2 * l.sc <= TH) team *= 2;
    for (int c0 = 0; c0 < l.sc; c0 += TH / team) {
        const int c = c0 + tid / team;
        double a = 0., q = 0.;
        if (c < l.sc)
            for (int i = tid & (team - 1); i < rows; i += team) {
                const float2 v = red[i * l.sc + c];
                a += v.x;
                q += v.y;
            }
        for (int o = team >> 1; o; o >>= 1) {
            a += shfl_xor_d(a, o);
            q += shfl_xor_d(q, o);
        }
        if (c < l.sc && (tid & (team - 1)) == 0) {
            const int cc = l.ch0 + c;
            const double f = p.ss ? 1. + (double)p.ss[(size_t)b * p.ld_ss + cc] : 1., w = f * p.gamma[cc];
            ch[c] = make_double2(w * a, w * q);
            put_dss(p, b, cc, a, q);
            if (p.B == 1) {   // nothing to sum over: the affine's gradient is complete
                p.dgamma[cc] = (float)(f * q);
                p.dbeta[cc] = (float)(f * a);
            } else {
                p.csum[(size_t)b * p.C + cc] = make_float2((float)a, (float)q);
            }
        }
    }
    __syncthreads();
    group_items<TH>(l.sc / cg, cg, tid, scratch, [&](int g, int i) { return ch[g * cg + i]; },
                   [&](int g, double s, double q) { gm[g] = make_float2((float)(s * p.inv_n), (float)(q * p.inv_n)); });
    if (k <= 0) return;
    float u1[V], u2[V];
    each_group<V>(l.cv * V, cg, [&](int j, int g) {
        u1[j] = co.r[j] * gm[g].x;
        u2[j] = co.r[j] * co.r[j] * gm[g].y;
    });
    bwd_emit<GN_R>(bx, bd, co, u1, u2, (T*)p.out + (size_t)b * p.n * p.ldo + cb, p.ldo, l.rl, l.RL, k, silu);
}

// ---------------------------------------------------------------------------------------- launch rules
int gcd_i(int a, int b) { return b ? gcd_i(b, a % b) : a; }

// channels a block owns: whole groups and whole vectors, at least `bytes` of a row
int slab_channels(int C, int cg, int V, int es, int bytes) {
    const int unit = cg / gcd_i(cg, V) * V;
    int s = unit;
    while (s * es < bytes && s < C) s += unit;
    return s < C ? s : C;
}

size_t resident_lds(int T, int slab, int cg, int V) {
    return (size_t)T * V * 8 + (size_t)T / 64 * 16 + (size_t)slab * 16 + (size_t)(slab / cg) * 8;
}

// threads of the resident form (0: the slab's rows do not fit the registers of a block, or its sums 64 KB of LDS)
int resident_threads(int n, int slab, int cg, int V) {
    const int tw = slab / V;
    for (int T = 256; T <= 512; T *= 2)
        if (tw <= T && (long long)(T / tw) * GN_R >= n && resident_lds(T, slab, cg, V) <= 65536) return T;
    return 0;
}

// row chunks of the streamed form: one block per CU over the whole launch (a block's way through its statistics costs about
// 3 us whatever its rows: 8 x 64 x 64 x 256 bf16 15.0 us with one, 16.7 with two, 22.9 with four), 16 rows at least.  The
// workspace counts a single slab: an upper bound that does not depend on vector width, and so not on alignment.
int stream_chunks(int B, int n, int slabs) {
    long long c = 256 / ((long long)B * slabs);
    c = c < 1 ? 1 : (c > GN_MAX_CHUNKS ? GN_MAX_CHUNKS : c);
    const int most = ceil_div(n, 16);
    return c < most ? (int)c : most;
}

size_t al256(size_t v) { return (v + 255) & ~(size_t)255; }

// a slab of more vectors than a block has threads must be a single group (the kernels' wide path)
bool slab_ok(int C, int cg, int V, int es) {
    const int s = slab_channels(C, cg, V, es, 128);
    return s / V <= GN_T || s == cg;
}

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

// What the second pass reads again was read by the first: where rows in and out together near the size of the memory-side cache (256 MB),
// written rows would drive out rows still to come, so they go past it (16 x 256 x 256 x 64 bf16: 87 -> 74 us).
bool bypass_caches(const GnArgs& p, size_t row_bytes) { return (size_t)p.B * p.n * row_bytes > ((size_t)192 << 20); }

void stream_shape(GnArgs& p, int V, int es) {
    p.slab = slab_channels(p.C, p.cg, V, es, 128);
    p.chunks = stream_chunks(p.B, p.n, ceil_div(p.C, p.slab));
    p.rows = ceil_div(p.n, p.chunks);
}

template <typename TX, typename TO, int V> void launch_fwd(GnArgs p, hipStream_t st) {
    const int es = sizeof(TX);
    p.slab = slab_channels(p.C, p.cg, V, es, 64);
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
    stream_shape(p, V, es);
    const dim3 grid(p.chunks, ceil_div(p.C, p.slab), p.B);
    const size_t scratch = GN_T / 64 * 16;
    hipLaunchKernelGGL((gn_stats_kernel<TX, V>), grid, dim3(GN_T), scratch + (size_t)GN_T * (V > 2 ? V : 2) * 8, st, p);
    const size_t lds = scratch + (size_t)(p.slab / p.cg) * 8;
    if (bypass_caches(p, (size_t)p.C * (sizeof(TX) + sizeof(TO))))
        hipLaunchKernelGGL((gn_apply_kernel<TX, TO, V, true>), grid, dim3(GN_T), lds, st, p);
    else
        hipLaunchKernelGGL((gn_apply_kernel<TX, TO, V, false>), grid, dim3(GN_T), lds, st, p);
}

template <typename T, int V> void launch_bwd(GnArgs p, hipStream_t st) {
    p.slab = slab_channels(p.C, p.cg, V, sizeof(T), 64);
    const int TH = resident_threads(p.n, p.slab, p.cg, V);
    if (TH) {
        const size_t lds = resident_lds(TH, p.slab, p.cg, V);
        const dim3 grid(ceil_div(p.C, p.slab), p.B);
        p.sums = p.csum;
        p.sum_chunks = 1;
        if (TH == 256)
            hipLaunchKernelGGL((gn_bwd_resident_kernel<T, V, 256>), grid, dim3(256), lds, st, p);
        else
            hipLaunchKernelGGL((gn_bwd_resident_kernel<T, V, 512>), grid, dim3(512), lds, st, p);
        if (p.B > 1) hipLaunchKernelGGL(gn_bwd_affine_kernel, dim3(ceil_div(p.C, 64)), dim3(GN_T), 0, st, p);
        return;
    }
    stream_shape(p, V, sizeof(T));
    const int slabs = ceil_div(p.C, p.slab);
    hipLaunchKernelGGL((gn_bwd_sums_kernel<T, V>), dim3(p.chunks, slabs, p.B), dim3(GN_T),
                       (size_t)GN_T * V * 8 + (size_t)p.slab * 16, st, p);
    p.sums = p.cpart;
    p.sum_chunks = p.chunks;
    if (p.slab * p.chunks > 8192) {   // 64 KB of partials a block: sum them once instead
        hipLaunchKernelGGL(gn_bwd_reduce_kernel, dim3(ceil_div(p.C, 64), p.B), dim3(GN_T), 0, st, p);
        p.sums = p.csum;
        p.sum_chunks = 1;
    }
    // 8 KB of it serve the blocks that form dgamma and dbeta
    const size_t lds = GN_T / 64 * 16 + (size_t)(p.slab > GN_T ? p.slab : GN_T) * 16 + (size_t)(p.slab / p.cg) * 8;
    const dim3 grid(p.chunks, slabs, p.B + 1);
    if (bypass_caches(p, (size_t)p.C * sizeof(T) * 3))
        hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, true>), grid, dim3(GN_T), lds, st, p);
    else
        hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, false>), grid, dim3(GN_T), lds, st, p);
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

// A range of memory that a call reads or writes beside its rows.
struct Range {
    const void* p;
    size_t n;
    const char* name;
};
size_t ss_bytes(size_t ld, int B, int C) { return ((size_t)(B - 1) * ld + 2 * (size_t)C) * 4; }

// Vectors are read again after others have been written: none that is written may meet another operand.  First `written` of all.
int check_apart(const char* what, const Range* all, int written, int count) {
    for (int i = 0; i < written; ++i)
        for (int j = i + 1; j < count; ++j)
            UWIR_CHECK(!all[i].p || !all[j].p || !overlaps(all[i].p, all[i].n, all[j].p, all[j].n), "%s: %s overlaps %s", what,
                       all[i].name, all[j].name);
    return UWIR_OK;
}

int check_common(const char* what, int B, int n, int C, int G, int act, size_t workspace_bytes) {
    // row indexes are 32 bits, and a thread looks up to 4 rows of each of GN_T lanes ahead
    UWIR_CHECK(B > 0 && B <= 65534 && n > 0 && n < (1 << 30) && C > 0 && C <= GN_MAX_C,
               "%s: bad shape (0 < B <= 65534, 0 < n < 2^30, 0 < C <= %d)", what, GN_MAX_C);
    UWIR_CHECK(G > 0 && C % G == 0, "%s: groups must divide C", what);
    UWIR_CHECK(act == UWIR_ACT_NONE || act == UWIR_ACT_SILU, "%s: act must be UWIR_ACT_NONE or UWIR_ACT_SILU", what);
    UWIR_CHECK(workspace_bytes >= uwir_group_norm_act_workspace_bytes(B, n, C, G), "%s: workspace too small", what);
    return UWIR_OK;
}

}  // namespace

// partials of the streamed form: per chunk and group (forward) or per chunk and channel (backward), and per image and channel
extern "C" size_t uwir_group_norm_act_workspace_bytes(int B, int n, int C, int groups) {
    if (B <= 0 || n <= 0 || C <= 0 || groups <= 0) return 0;
    const size_t ch = stream_chunks(B, n, 1);   // fewer with several slabs
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
    const size_t nc = (size_t)C * 4, ng = (size_t)B * groups * 4;
    const Range all[] = {{workspace, uwir_group_norm_act_workspace_bytes(B, n, C, groups), "the workspace"}, {mean, ng, "mean"}, {rstd, ng, "rstd"},
                         {out, bo, "out"}, {gamma, nc, "gamma"}, {beta, nc, "beta"}, {scale_shift, ss_bytes(ld_ss, B, C), "scale_shift"}, {x, bx, "x"}};
    if (int rc = check_apart("group_norm_act", all, 3, 8)) return rc;
    if (int rc = check_apart("group_norm_act", all + 3, 1, 4)) return rc;
    GnArgs p = {};
    p.x = x; p.out = out; p.gamma = gamma; p.beta = beta; p.ss = scale_shift; p.mean = mean; p.rstd = rstd;
    p.part = (double2*)workspace;
    p.ldx = ldx; p.ldo = ldo; p.ld_ss = ld_ss;
    p.B = B; p.n = n; p.C = C; p.G = groups; p.cg = C / groups; p.eps = eps; p.act = act; p.inv_n = 1. / ((double)n * p.cg);
    // widest vector (16 bytes of x at most) that the channel count, strides and addresses allow
    int V = 16 / ex;
    while (V > 1 && (C % V || !slab_ok(C, p.cg, V, ex) || !vec_ok(x, ldx, V, ex) || !vec_ok(out, ldo, V, eo))) V >>= 1;
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
    const size_t nc = (size_t)C * 4, ng = (size_t)B * groups * 4;
    const Range all[] = {{workspace, uwir_group_norm_act_workspace_bytes(B, n, C, groups), "the workspace"},
                         {dgamma, nc, "dgamma"}, {dbeta, nc, "dbeta"}, {dscale_shift, ss_bytes(ld_dss, B, C), "dscale_shift"},
                         {dx, bo, "dx"}, {gamma, nc, "gamma"}, {beta, nc, "beta"}, {mean, ng, "mean"}, {rstd, ng, "rstd"},
                         {scale_shift, ss_bytes(ld_ss, B, C), "scale_shift"}, {x, bx, "x"}, {dy, by, "dy"}};
    if (int rc = check_apart("group_norm_act_backward", all, 4, 12)) return rc;
    if (int rc = check_apart("group_norm_act_backward", all + 4, 1, 6)) return rc;
    GnArgs p = {};
    p.x = x; p.dy = dy; p.out = dx; p.gamma = gamma; p.beta = beta; p.ss = scale_shift; p.mean_in = mean; p.rstd_in = rstd;
    p.dgamma = dgamma; p.dbeta = dbeta; p.dss = dscale_shift;
    p.ldx = ldx; p.ldy = ldy; p.ldo = ldd; p.ld_ss = ld_ss; p.ld_dss = ld_dss;
    p.B = B; p.n = n; p.C = C; p.G = groups; p.cg = C / groups; p.act = act; p.inv_n = 1. / ((double)n * p.cg);
    p.cpart = (float2*)workspace;
    p.csum = (float2*)((char*)workspace + al256((size_t)B * stream_chunks(B, n, 1) * C * 8));
    int V = 16 / es;
    while (V > 1 && (C % V || !slab_ok(C, p.cg, V, es) || !vec_ok(x, ldx, V, es) || !vec_ok(dy, ldy, V, es) || !vec_ok(dx, ldd, V, es))) V >>= 1;
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
