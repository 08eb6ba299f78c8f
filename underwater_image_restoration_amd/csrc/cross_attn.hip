// Cross attention of image rows to an encoder's states, forward: one pass over the keys with a running maximum and sum.
//
// The rows of all query heads that share a key head are packed into one row axis (R = nq * heads / kv_heads rows per
// image and key head), so shared heads read their keys once.  S^T = K q^T puts a query row on a lane and its keys on the
// accumulator's registers: maximum and sum are register reductions plus one exchange between the wave's halves, and
// P feeds O^T += V^T P from registers (cross_attn.h).
//   tile kernel   4 waves x 32 QG rows share key tiles in LDS
//   row kernel    R <= 32: the 4 waves take key tiles of their own and join at the end
// Either may split the key axis over blocks when there are few rows; a second launch joins the parts.
// The running maximum is only raised when a lane's sum over a unit passes 2^16: until then the probabilities of the maximum held
// are exact enough (fp32 keeps its 24 bits at any exponent), and the usual tile pays no rescale.  Probabilities are rounded to bf16
// for the second product (2^-8 of each at most), their sum is that of the unrounded ones.
#include "cross_attn.h"

#include <utility>

using namespace xattn;

namespace {

struct XArgs {
    const void *q, *k, *v;
    void* o;
    float* lse;
    const int* lens;
    const unsigned char* mask;
    float* part_o;      // split: [splits][B * KV * R][hd] normalised outputs
    float* part_l;      // [splits][B * KV * R] log2-domain normalisers (-inf: nothing seen)
    size_t ldq, ldk, ldv, ldo, ldm;
    int B, nq, nk, H, KV, hd, G, R, splits, nblocks, qtiles;
    Divisor by_g;
    float c;            // scale * log2(e)
    float m0;           // the running reference before any key is seen: low, and m0 * c finite
};

// One 32-row group of a wave: running maximum m (raw scores), this lane's part of the sum, O^T.
template <typename T, int HD> struct Group {
    typedef Mma<T> M;
    static constexpr int KS = HD / M::KSTEP, DG = HD / 32;
    typename M::frag q[KS];
    f32x16 o[DG];
    float m, l;

    __device__ __forceinline__ void init(const XArgs& p, int b, int kv, int r, int lane) {
        const bool ok = r < p.R;
        const RowRef f = row_ref(p, b, kv, ok ? r : 0);
        const T* src = (const T*)p.q + f.row * p.ldq + (size_t)f.head * p.hd;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int d = ks * M::KSTEP + (lane >> 5) * M::VEC;
            if (ok && d < p.hd)
                q[ks] = *reinterpret_cast<const typename M::frag*>(src + d);
            else
#pragma unroll
                for (int j = 0; j < M::VEC; ++j) q[ks][j] = (T)0.f;
        }
#pragma unroll
        for (int g = 0; g < DG; ++g) zero16(o[g]);
        m = p.m0;
        l = 0.f;
    }

    // Scores s of 32 keys -> probabilities relative to the running reference m.  m need not be the maximum, only near enough for
    // the fp32 range: the probabilities are formed first, and only where a lane's sum leaves 2^16 is the true maximum taken, the
    // output rescaled and the unit formed again.  A reference below the maximum costs no accuracy; what underflows next to it is
    // below 2^-120 of a sum that is at least 1; and the output before its division stays below nk 2^12 max |v|.
    // The first unit with a visible key does so by itself: m starts at m0, half the fp32 range below zero in scores and in their
    // products with c, so that visible scores lie far above it and hidden ones far below, and a unit without a visible key leaves
    // it there, with probabilities of 0.
    static __device__ __forceinline__ bool out_of_range(float sum) { return sum > 65536.f; }
    __device__ __forceinline__ void rescale(const f32x16& s, float c, typename M::Prob& pb, float& sum) {
        float mx = fmaxf(s[0], s[1]);
#pragma unroll
        for (int r = 2; r < 16; r += 2) mx = fmaxf(fmaxf(mx, s[r]), s[r + 1]);
        const float2 h = both_halves(mx);
        const float mn = fmaxf(m, fmaxf(h.x, h.y)), f = __builtin_amdgcn_exp2f((m - mn) * c);
        m = mn;
        l *= f;
#pragma unroll
        for (int g = 0; g < DG; ++g)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[g][r] *= f;
        pb = form(s, c, sum);
    }
    // the sum is that of the unrounded probabilities: lse keeps fp32's accuracy
    __device__ __forceinline__ typename M::Prob form(const f32x16& s, float c, float& sum) const {
        const float mc = m * c;
        float pr[16], l0 = 0.f, l1 = 0.f;
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
            pr[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -mc));
            pr[r + 1] = __builtin_amdgcn_exp2f(fmaf(s[r + 1], c, -mc));
            l0 += pr[r];
            l1 += pr[r + 1];
        }
        sum = l0 + l1;
        return M::pack(pr);
    }
};

// out and lse of one lane's row, or its part of a split
template <typename T, int HD>
__device__ __forceinline__ void write_row(const XArgs& p, int b, int kv, int split, int r, int lane, const f32x16* o, float l, float m) {
    if (r >= p.R) return;
    const float inv = l > 0.f ? __builtin_amdgcn_rcpf(l) : 0.f;   // 1 ulp
    const float l2 = l > 0.f ? fmaf(m, p.c, __builtin_amdgcn_logf(l)) : -INFINITY;   // v_log_f32: base 2
    const RowRef f = row_ref(p, b, kv, r);
    if (p.splits > 1) {
        const size_t pr = ((size_t)split * p.B * p.KV + (size_t)b * p.KV + kv) * p.R + r;
        if (lane < 32) p.part_l[pr] = l2;
        float* dst = p.part_o + pr * p.hd;
#pragma unroll
        for (int g = 0; g < HD / 32; ++g)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                float v[8];
                gather8(o[g], t, v);
                const int d = 32 * g + 16 * t + 8 * (lane >> 5);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] *= inv;
                if (d < p.hd) store8(dst + d, v);
            }
        return;
    }
    if (p.lse && lane < 32) p.lse[((size_t)b * p.H + f.head) * p.nq + (f.row - (size_t)b * p.nq)] = l2 * LN2;
    T* dst = (T*)p.o + f.row * p.ldo + (size_t)f.head * p.hd;
#pragma unroll
    for (int g = 0; g < HD / 32; ++g)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            float v[8];
            gather8(o[g], t, v);
            const int d = 32 * g + 16 * t + 8 * (lane >> 5);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= inv;
            if (d < p.hd) store8(dst + d, v);
        }
}

// keys [begin, end) of this block's part; parts are multiples of `unit` keys of the image's own length
__device__ __forceinline__ void key_range(const XArgs& p, int b, int split, int unit, int& begin, int& end) {
    int len = p.nk;
    if (p.lens) len = max(0, min(p.nk, p.lens[b]));
    if (p.splits == 1) {
        begin = 0;
        end = len;
        return;
    }
    const int tiles = (len + unit - 1) / unit, per = (tiles + p.splits - 1) / p.splits;
    begin = min(len, split * per * unit);
    end = min(len, (split + 1) * per * unit);
}

// NW waves x 32 QG rows share key tiles of KT keys in LDS (two buffers, the next tile loading meanwhile).  Nothing in a wave's way
// through a tile overlaps its matrix and its vector work (scores, probabilities, output); the waves of a SIMD do.  With two row
// groups a wave reads every fragment of K and V from LDS once for both: LDS, not arithmetic, held the one-group form back.
// Bound: 8 x 128 x 128 queries over 577 states, 8 heads of 64, 235 us = 660 TF of 4 hd flops a pair.  A 32 x 32 unit takes 463
// cycles of a SIMD to issue its vector work (384: 16 exp at 8, the scale, the sum, the rounding) and its 18 matrix instructions,
// which keep the matrix pipe for 288 (both counted); and 50 us of reading q and writing out, which the blocks of a CU, equal and started together, do at the same time.
// 8 x 32 x 32 over 50 states, 8 heads of 32: 5.9 us, latency.  fp32: one wave a SIMD at most, exact fp32 MFMA; 2 x 32 x 32 over
// 197, 16 heads of 32, 16 us.
template <typename T, int HD, int NW, int QG>
__global__ void __launch_bounds__(NW * 64, QG == 2 ? 2 : 1) xattn_tile_kernel(XArgs p) {
    typedef Tile<T, HD> L;
    typedef typename L::M M;
    typedef typename M::frag frag;
    constexpr int TH = NW * 64, KT = 64, NC = KT * L::CPR / TH < 1 ? 1 : KT * L::CPR / TH;   // 16-byte chunks per thread and tile
    static_assert(KT * L::CPR % TH == 0 || KT * L::CPR < TH, "whole chunks per thread");
    __shared__ __attribute__((aligned(16))) T sK[2][KT * L::STR];
    __shared__ __attribute__((aligned(16))) T sV[2][KT * L::STR];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned vid = xcd_order(blockIdx.x, p.nblocks);
    const Item it = block_item(vid, p.KV, p.B, p.splits, p.qtiles, p.lens != nullptr);
    const int b = it.b, kv = it.kv, split = it.part, qt = it.tile;
    int begin, end;
    key_range(p, b, split, KT, begin, end);

    const T* K = (const T*)p.k + (size_t)b * p.nk * p.ldk + (size_t)kv * p.hd;
    const T* V = (const T*)p.v + (size_t)b * p.nk * p.ldv + (size_t)kv * p.hd;
    const unsigned char* mask = p.mask ? p.mask + (size_t)b * p.ldm : nullptr;
    const int width = p.hd * (int)sizeof(T);
    const size_t ldkb = p.ldk * sizeof(T), ldvb = p.ldv * sizeof(T);
    const bool loads = KT * L::CPR >= TH || tid < KT * L::CPR;
    unsigned ko[NC], vo[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int row = (tid + TH * i) / L::CPR, col = (tid + TH * i) % L::CPR * 16;
        ko[i] = tile_offset(row, (unsigned)ldkb, col, width);
        vo[i] = tile_offset(row, (unsigned)ldvb, col, width);
    }
    frag rk[NC], rv[NC];
    bool vis;
    auto load = [&](int k0) {
        const __amdgpu_buffer_rsrc_t kr = tile_buffer(K, ldkb, k0, end, width), vr = tile_buffer(V, ldvb, k0, end, width);
        if (loads) {
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                rk[i] = buffer_frag<frag>(kr, ko[i]);
                rv[i] = buffer_frag<frag>(vr, vo[i]);
            }
        }
        vis = k0 + lane < end && (!mask || mask[k0 + lane]);
    };
    // keys hidden by the mask enter as zeros: what they hold (NaN included) must not meet the zero probabilities
    auto store = [&](int buf, unsigned long long bits) {
        if (!loads) return;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int row = (tid + TH * i) / L::CPR, d = (tid + TH * i) % L::CPR * L::VEC;
            if (mask && !((bits >> row) & 1)) rk[i] = rv[i] = frag{};
            *reinterpret_cast<frag*>(&sK[buf][row * L::STR + d]) = rk[i];
            *reinterpret_cast<frag*>(&sV[buf][row * L::STR + d]) = rv[i];
        }
    };

    Group<T, HD> gr[QG];
    const int first = (qt * NW + wave) * 32 * QG, row0 = first + (lane & 31);
#pragma unroll
    for (int g = 0; g < QG; ++g) gr[g].init(p, b, kv, row0 + 32 * g, lane);
    const float c = p.c;
    const bool idle = first >= p.R;   // the whole wave lies behind the last row: it only helps to load

    unsigned long long bits = 0;
    if (begin < end) {
        load(begin);
        bits = __ballot(vis);
        store(0, bits);
    }
    __syncthreads();
    int buf = 0;
    for (int k0 = begin; k0 < end; k0 += KT, buf ^= 1) {
        const bool more = k0 + KT < end;
        if (more) load(k0 + KT);
        if (bits && !idle) {
#pragma unroll
            for (int kb = 0; kb < KT / 32; ++kb) {
                f32x16 s[QG];
#pragma unroll
                for (int g = 0; g < QG; ++g) zero16(s[g]);
                const T* kr = &sK[buf][(32 * kb + (lane & 31)) * L::STR + (lane >> 5) * L::VEC];
#pragma unroll
                for (int ks = 0; ks < Group<T, HD>::KS; ++ks) {
                    const frag kf = *reinterpret_cast<const frag*>(kr + ks * M::KSTEP);
#pragma unroll
                    for (int g = 0; g < QG; ++g) M::rows(s[g], kf, gr[g].q[ks]);
                }
                const auto hider = M::hider(!(((unsigned)(bits >> (32 * kb)) >> (lane & 31)) & 1), lane);
#pragma unroll
                for (int g = 0; g < QG; ++g) M::hide(s[g], hider, lane);
                typename M::Prob pb[QG];
                float sum[QG];
                bool far = false;
#pragma unroll
                for (int g = 0; g < QG; ++g) {
                    pb[g] = gr[g].form(s[g], c, sum[g]);
                    far |= gr[g].out_of_range(sum[g]);
                }
                if (__any(far))
#pragma unroll
                    for (int g = 0; g < QG; ++g) gr[g].rescale(s[g], c, pb[g], sum[g]);
#pragma unroll
                for (int g = 0; g < QG; ++g) gr[g].l += sum[g];
#pragma unroll
                for (int dg = 0; dg < HD / 32; ++dg) {
                    const auto vf = M::template col_frags<L::STR>(&sV[buf][32 * kb * L::STR + 32 * dg], lane);
#pragma unroll
                    for (int g = 0; g < QG; ++g) M::cols(gr[g].o[dg], vf, pb[g]);
                }
            }
        }
        if (more) {
            bits = __ballot(vis);
            store(buf ^ 1, bits);
        }
        __syncthreads();
    }
#pragma unroll
    for (int g = 0; g < QG; ++g) {
        const float2 h = both_halves(gr[g].l);
        write_row<T, HD>(p, b, kv, split, row0 + 32 * g, lane, gr[g].o, h.x + h.y, gr[g].m);
    }
}

// R <= 32 rows: every wave walks key tiles of 32 of its own (LDS private to the wave, no block barrier in the loop).
// Bound by reading k and v once: 16 images, one query of 32 heads over up to 8192 states of 8 heads of 64 (142 MB at these lengths)
// 42 us with the join (6 us) from HBM, 3.4 TB/s; with one length for all images 60 us (268 MB, 4.5 TB/s): the rest is the long
// images' parts ending last.
template <typename T, int HD>
__global__ void __launch_bounds__(256) xattn_row_kernel(XArgs p) {
    typedef Tile<T, HD> L;
    typedef typename L::M M;
    constexpr int KT = 32, NC = KT * L::CPR / 64;
    constexpr int TILE = KT * L::STR;
    constexpr int JOIN = 4 * 32 * (HD + 1) * 4, LOOP = 4 * 2 * TILE * (int)sizeof(T);
    __shared__ __attribute__((aligned(16))) char smem[JOIN > LOOP ? JOIN : LOOP];
    __shared__ float sm[4][32], sl[4][32];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    T* sK = reinterpret_cast<T*>(smem) + wave * 2 * TILE;
    T* sV = sK + TILE;
    const unsigned vid = xcd_order(blockIdx.x, p.nblocks);
    const Item it = block_item(vid, p.KV, p.B, p.splits, 1, p.lens != nullptr);
    const int b = it.b, kv = it.kv, split = it.part;
    int begin, end;
    key_range(p, b, split, 4 * KT, begin, end);
    const T* K = (const T*)p.k + (size_t)b * p.nk * p.ldk + (size_t)kv * p.hd;
    const T* V = (const T*)p.v + (size_t)b * p.nk * p.ldv + (size_t)kv * p.hd;
    const unsigned char* mask = p.mask ? p.mask + (size_t)b * p.ldm : nullptr;

    typename M::frag rk[NC], rv[NC];
    bool vis;
    auto load = [&](int k0) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int ci = lane + 64 * i, d = (ci % L::CPR) * L::VEC, key = min(k0 + ci / L::CPR, end - 1);
            if (d < p.hd) {
                rk[i] = *reinterpret_cast<const typename M::frag*>(K + (size_t)key * p.ldk + d);
                rv[i] = *reinterpret_cast<const typename M::frag*>(V + (size_t)key * p.ldv + d);
            } else {
#pragma unroll
                for (int j = 0; j < L::VEC; ++j) rk[i][j] = rv[i][j] = (T)0.f;
            }
        }
        const int key = k0 + (lane & 31);
        vis = key < end && (!mask || mask[key]);
    };

    Group<T, HD> gr;
    gr.init(p, b, kv, lane & 31, lane);
    const float c = p.c;
    int k0 = begin + wave * KT;
    if (k0 < end) load(k0);
    for (; k0 < end; k0 += 4 * KT) {
        const unsigned bits = (unsigned)__ballot(vis);
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int ci = lane + 64 * i, row = ci / L::CPR, d = (ci % L::CPR) * L::VEC;
            if (bits != ~0u && !((bits >> row) & 1)) {
#pragma unroll
                for (int j = 0; j < L::VEC; ++j) rk[i][j] = rv[i][j] = (T)0.f;
            }
            *reinterpret_cast<typename M::frag*>(sK + row * L::STR + d) = rk[i];
            *reinterpret_cast<typename M::frag*>(sV + row * L::STR + d) = rv[i];
        }
        // the wave's own LDS operations stay in order; only the compiler has to be held
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (k0 + 4 * KT < end) load(k0 + 4 * KT);
        if (bits) {
            f32x16 s;
            zero16(s);
            const T* kr = sK + (lane & 31) * L::STR + (lane >> 5) * L::VEC;
#pragma unroll
            for (int ks = 0; ks < Group<T, HD>::KS; ++ks)
                M::rows(s, *reinterpret_cast<const typename M::frag*>(kr + ks * M::KSTEP), gr.q[ks]);
            M::hide(s, M::hider(!((bits >> (lane & 31)) & 1), lane), lane);
            float sum;
            typename M::Prob pb = gr.form(s, c, sum);
            if (__any(gr.out_of_range(sum))) gr.rescale(s, c, pb, sum);
            gr.l += sum;
#pragma unroll
            for (int dg = 0; dg < HD / 32; ++dg) M::template cols<L::STR>(gr.o[dg], sV + 32 * dg, lane, pb);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    // join the four waves: common maximum, scaled sums
    const float2 h = both_halves(gr.l);
    if (lane < 32) {
        sm[wave][lane] = gr.m;
        sl[wave][lane] = h.x + h.y;
    }
    __syncthreads();   // also: every wave is done with its tiles, smem becomes the outputs' buffer
    float m = p.m0, l = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) m = fmaxf(m, sm[w][lane & 31]);
#pragma unroll
    for (int w = 0; w < 4; ++w) l += sl[w][lane & 31] * __builtin_amdgcn_exp2f((sm[w][lane & 31] - m) * c);
    const float f = __builtin_amdgcn_exp2f((gr.m - m) * c);
    float* so = reinterpret_cast<float*>(smem);   // [wave][row][HD + 1]
#pragma unroll
    for (int dg = 0; dg < HD / 32; ++dg)
#pragma unroll
        for (int r = 0; r < 16; ++r)
            so[(wave * 32 + (lane & 31)) * (HD + 1) + 32 * dg + (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5)] = gr.o[dg][r] * f;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int dg = 0; dg < HD / 32; ++dg)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float a = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w)
                a += so[(w * 32 + (lane & 31)) * (HD + 1) + 32 * dg + (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5)];
            gr.o[dg][r] = a;
        }
    write_row<T, HD>(p, b, kv, split, lane & 31, lane, gr.o, l, m);
}

// out = sum_i 2^(l_i - L) o_i over the parts; one thread per row and 8 columns
template <typename T>
__global__ void __launch_bounds__(256) xattn_join_kernel(XArgs p) {
    const int cpr = p.hd / 8;
    const size_t rows = (size_t)p.B * p.KV * p.R, i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= rows * cpr) return;
    const size_t pr = i / cpr;
    const int d = 8 * (int)(i % cpr);
    float m = -INFINITY;
#pragma unroll 8
    for (int s = 0; s < p.splits; ++s) m = fmaxf(m, p.part_l[s * rows + pr]);
    float l = 0.f, v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
    if (m > -INFINITY)
#pragma unroll 8
        for (int s = 0; s < p.splits; ++s) {   // eight parts' loads under way at a time
            const float w = __builtin_amdgcn_exp2f(p.part_l[s * rows + pr] - m);
            const float* src = p.part_o + (s * rows + pr) * p.hd + d;
            const f32x4 a = *reinterpret_cast<const f32x4*>(src), e = *reinterpret_cast<const f32x4*>(src + 4);
            l += w;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[j] = fmaf(w, a[j], v[j]);
                v[4 + j] = fmaf(w, e[j], v[4 + j]);
            }
        }
    const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= inv;
    const int r = (int)(pr % p.R), kv = (int)(pr / p.R % p.KV), b = (int)(pr / p.R / p.KV);
    const RowRef f = row_ref(p, b, kv, r);
    store8((T*)p.o + f.row * p.ldo + (size_t)f.head * p.hd + d, v);
    if (p.lse && d == 0)
        p.lse[((size_t)b * p.H + f.head) * p.nq + (f.row - (size_t)b * p.nq)] = l > 0.f ? (m + __builtin_amdgcn_logf(l)) * LN2 : -INFINITY;
}

// ---------------------------------------------------------------------------------------- launch rules
struct Plan {
    bool row;       // row kernel
    bool two;       // two row groups a wave
    int qtiles, splits;
};

Plan plan_fwd(int B, int nq, int nk, int H, int KV, int hd, int dtype) {
    Plan pl = {};
    const long long R = (long long)nq * (H / KV), bk = (long long)B * KV;
    pl.row = R <= 32;
    pl.two = false;
    long long blocks;
    const int unit = 256;   // smallest part worth a block of its own
    if (pl.row) {
        pl.qtiles = 1;
        blocks = bk;
    } else {
        // where 256 rows a block still give every CU two blocks (bf16; the registers of 128 columns leave no room)
        pl.two = dtype == UWIR_BF16 && hd <= 64 && R > 128 && (R + 255) / 256 * bk >= 512;
        const int rows = pl.two ? 256 : 128;
        pl.qtiles = (int)((R + rows - 1) / rows);
        blocks = bk * pl.qtiles;
    }
    // few blocks: parts of the key axis until every CU has two blocks (four of the row kernel, which only streams)
    const int want = pl.row ? 1024 : 512;
    long long s = blocks >= 384 ? 1 : (want + blocks - 1) / (blocks > 0 ? blocks : 1);
    const long long most = nk / unit;
    if (s > most) s = most;
    if (s > 64) s = 64;
    pl.splits = s < 1 ? 1 : (int)s;
    return pl;
}

template <typename T, int HD> void launch(const XArgs& p, const Plan& pl, hipStream_t st) {
    if (pl.row)
        hipLaunchKernelGGL((xattn_row_kernel<T, HD>), dim3(p.nblocks), dim3(256), 0, st, p);
    else if (pl.two) {
        if constexpr (sizeof(T) == 2 && HD <= 64)
            hipLaunchKernelGGL((xattn_tile_kernel<T, HD, 4, 2>), dim3(p.nblocks), dim3(256), 0, st, p);
    } else
        hipLaunchKernelGGL((xattn_tile_kernel<T, HD, 4, 1>), dim3(p.nblocks), dim3(256), 0, st, p);
    if (p.splits > 1) {
        const size_t n = (size_t)p.B * p.KV * p.R * (p.hd / 8);
        hipLaunchKernelGGL((xattn_join_kernel<T>), dim3((unsigned)ceil_div_sz(n, 256)), dim3(256), 0, st, p);
    }
}

}  // namespace

extern "C" size_t uwir_cross_attn_workspace_bytes(int B, int nq, int nk, int heads, int kv_heads, int hd, int dtype) {
    if (B <= 0 || nq <= 0 || nk <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || hd <= 0) return 0;
    const Plan pl = plan_fwd(B, nq, nk, heads, kv_heads, hd, dtype);
    if (pl.splits == 1) return 0;
    const size_t rows = (size_t)pl.splits * B * heads * nq;
    return al256(rows * hd * 4) + al256(rows * 4);
}

extern "C" int uwir_cross_attn(const void* q, size_t ldq, const void* k, size_t ldk, const void* v, size_t ldv, int dtype, int B,
                               int nq, int nk, int heads, int kv_heads, int hd, float scale, const int* key_lens,
                               const unsigned char* key_mask, size_t ld_mask, void* out, size_t ldo, float* lse, void* workspace,
                               size_t workspace_bytes, uwir_stream_t stream) {
    if (int rc = xattn_check("cross_attn", dtype, B, nq, nk, heads, kv_heads, hd, scale)) return rc;
    if (nq == 0) return UWIR_OK;
    const XMat in[] = {{q, ldq, heads, (size_t)B * nq, "q"}, {k, ldk, kv_heads, (size_t)B * nk, "k"}, {v, ldv, kv_heads, (size_t)B * nk, "v"}};
    const XMat res[] = {{out, ldo, heads, (size_t)B * nq, "out"}};
    if (int rc = xattn_check_mats("cross_attn", dtype, hd, in, 3, res, 1)) return rc;
    UWIR_CHECK(!key_mask || ld_mask >= (size_t)nk, "cross_attn: mask rows must have at least nk entries");
    const size_t need = uwir_cross_attn_workspace_bytes(B, nq, nk, heads, kv_heads, hd, dtype);
    UWIR_CHECK(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
               "cross_attn: workspace too small or not 16-byte aligned");
    const size_t nl = (size_t)B * heads * nq * sizeof(float);
    for (const auto& m : {std::make_pair(in, 3), std::make_pair(res, 1)}) {
        if (int rc = xattn_check_apart("cross_attn", "the workspace", workspace, need, dtype, hd, m.first, m.second)) return rc;
        if (int rc = xattn_check_apart("cross_attn", "lse", lse, nl, dtype, hd, m.first, m.second)) return rc;
    }
    const uintptr_t w = (uintptr_t)workspace, l = (uintptr_t)lse;
    UWIR_CHECK(!need || !lse || w + need <= l || l + nl <= w, "cross_attn: the workspace overlaps lse");
    const XRange beside[] = {{workspace, need, "the workspace"}, {lse, nl, "lse"}};
    if (int rc = xattn_check_keys("cross_attn", key_lens, key_mask, ld_mask, B, nk, dtype, hd, res, 1, beside, 2)) return rc;
    const Plan pl = plan_fwd(B, nq, nk, heads, kv_heads, hd, dtype);
    XArgs p = {};
    p.q = q; p.k = k; p.v = v; p.o = out; p.lse = lse; p.lens = key_lens; p.mask = key_mask;
    p.ldq = ldq; p.ldk = ldk; p.ldv = ldv; p.ldo = ldo; p.ldm = ld_mask;
    p.B = B; p.nq = nq; p.nk = nk; p.H = heads; p.KV = kv_heads; p.hd = hd;
    p.G = heads / kv_heads; p.R = nq * p.G; p.splits = pl.splits; p.qtiles = pl.qtiles;
    const long long nb = (long long)B * kv_heads * pl.qtiles * pl.splits;
    UWIR_CHECK(nb < (1ll << 24), "cross_attn: too many rows for one launch");   // 2^32 threads
    p.nblocks = (int)nb;
    p.c = scale * LOG2E;
    p.m0 = p.c > 1.f ? -1.7e38f / p.c : -1.7e38f;
    p.by_g = make_divisor(p.G);
    if (need) {
        p.part_o = (float*)workspace;
        p.part_l = (float*)((char*)workspace + al256((size_t)pl.splits * B * heads * nq * hd * 4));
    }
    hipStream_t st = (hipStream_t)stream;
    switch (hd_class(hd) + (dtype == UWIR_BF16)) {
        case 32: launch<float, 32>(p, pl, st); break;
        case 33: launch<bf16_t, 32>(p, pl, st); break;
        case 64: launch<float, 64>(p, pl, st); break;
        case 65: launch<bf16_t, 64>(p, pl, st); break;
        case 128: launch<float, 128>(p, pl, st); break;
        default: launch<bf16_t, 128>(p, pl, st); break;
    }
    UWIR_LAUNCH_CHECK("cross_attn");
    return UWIR_OK;
}
