// Cross attention, backward.  With s = scale q k^T over the visible keys and p = exp(s - lse):
//   D = sum_d dout out,  dv = p^T dout,  dp = dout v^T,  ds = p (dp - D),  dq = scale ds k,  dk = scale ds^T q
// More than a few keys take two kernels, each of which keeps its result in registers and forms p again (7 products instead of
// the 5 that one kernel with both results would need; in exchange nothing is accumulated through memory in an order that
// changes):
//   rows kernel  a wave owns 32 packed rows (cross_attn.hip), walks the keys: S^T = K q^T, dP^T = V dout^T,
//                dq^T += K^T dS; also forms D (few bf16 keys: from p and dP) and hands (lse, D) to the next kernel in packed-row order
//   keys kernel  a wave owns 32 keys, walks the rows of all query heads that share them: S = q K^T, dP = dout V^T,
//                dv^T += dout^T P, dk^T += q^T dS -- the sum over shared heads and rows never leaves the registers
// Either splits its long axis over blocks when there are few; the parts (fp32) are then summed in order by a last launch.
#include "cross_attn.h"

using namespace xattn;

namespace {

struct BArgs {
    const void *q, *k, *v, *o, *go;
    const float* lse;
    void *dq, *dk, *dv;
    const int* lens;
    const unsigned char* mask;
    float2* ld;                    // [B * KV][R] (lse in the log2 domain, D)
    float *part_q, *part_k, *part_v;
    size_t ldq, ldk, ldv, ldo, ldg, ld_dq, ld_dk, ld_dv, ldm;
    int B, nq, nk, H, KV, hd, G, R;
    int qsplits, qtiles, qblocks;  // rows kernel
    int ksplits, ktiles, kblocks;  // keys kernel
    Divisor by_g;
    float c, scale;
};

__device__ __forceinline__ int image_len(const BArgs& p, int b) {
    return p.lens ? max(0, min(p.nk, p.lens[b])) : p.nk;
}

// ---------------------------------------------------------------------------------------- dq
// EXACT_D: D from p and dP instead of dout . out.  out is rounded to bf16, and over few keys that moves dq and dk by 0.001 of their
// norm (0.0004 over 1500), next to 0.0017 for their own rounding; a walk more over up to 256 keys is cheap.
// Bound by vector issue as the forward kernel is, with two products in and one out a unit: 4 x 64 x 64 queries over up to 2048 states of
// lengths of their own, 8 heads of 64 on 2 key heads, 104 us.
template <typename T, int HD, int QG, bool EXACT_D>
__global__ void __launch_bounds__(256, QG == 2 ? 2 : 1) xattn_dq_kernel(BArgs p) {
    typedef Tile<T, HD> L;
    typedef typename L::M M;
    typedef typename M::frag frag;
    constexpr int KT = 64, NC = KT * L::CPR / 256, KS = HD / M::KSTEP, DG = HD / 32;
    __shared__ __attribute__((aligned(16))) T sK[2][KT * L::STR];
    __shared__ __attribute__((aligned(16))) T sV[2][KT * L::STR];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned vid = xcd_order(blockIdx.x, p.qblocks);
    const Item it = block_item(vid, p.KV, p.B, p.qsplits, p.qtiles, p.lens != nullptr);
    const int b = it.b, kv = it.kv, split = it.part, qt = it.tile, bk = b * p.KV + kv;
    int begin = 0, end = image_len(p, b);
    if (p.qsplits > 1) {
        const int tiles = (end + KT - 1) / KT, per = (tiles + p.qsplits - 1) / p.qsplits;
        begin = min(end, split * per * KT);
        end = min(end, (split + 1) * per * KT);
    }
    const T* K = (const T*)p.k + (size_t)b * p.nk * p.ldk + (size_t)kv * p.hd;
    const T* V = (const T*)p.v + (size_t)b * p.nk * p.ldv + (size_t)kv * p.hd;
    const unsigned char* mask = p.mask ? p.mask + (size_t)b * p.ldm : nullptr;
    const int width = p.hd * (int)sizeof(T);
    const size_t ldkb = p.ldk * sizeof(T), ldvb = p.ldv * sizeof(T);
    unsigned ko[NC], vo[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int row = (tid + 256 * i) / L::CPR, col = (tid + 256 * i) % L::CPR * 16;
        ko[i] = tile_offset(row, (unsigned)ldkb, col, width);
        vo[i] = tile_offset(row, (unsigned)ldvb, col, width);
    }
    frag rk[NC], rv[NC];
    bool vis;
    auto load = [&](int k0) {
        const __amdgpu_buffer_rsrc_t kr = tile_buffer(K, ldkb, k0, end, width), vr = tile_buffer(V, ldvb, k0, end, width);
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            rk[i] = buffer_frag<frag>(kr, ko[i]);
            rv[i] = buffer_frag<frag>(vr, vo[i]);
        }
        vis = k0 + lane < end && (!mask || mask[k0 + lane]);
    };
    auto store = [&](int buf, unsigned long long bits) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int row = (tid + 256 * i) / L::CPR, d = (tid + 256 * i) % L::CPR * L::VEC;
            if (mask && !((bits >> row) & 1)) rk[i] = rv[i] = frag{};   // whatever keys hidden by the mask hold
            *reinterpret_cast<frag*>(&sK[buf][row * L::STR + d]) = rk[i];
            *reinterpret_cast<frag*>(&sV[buf][row * L::STR + d]) = rv[i];
        }
    };

    frag fq[QG][KS], fg[QG][KS];
    f32x16 dq[QG][DG];
    float l2[QG], D[QG];
    const int row0 = (qt * 4 + wave) * 32 * QG + (lane & 31);
#pragma unroll
    for (int g = 0; g < QG; ++g) {
        const int r = row0 + 32 * g;
        const bool ok = r < p.R;
        const RowRef f = row_ref(p, b, kv, ok ? r : 0);
        const T* Q = (const T*)p.q + f.row * p.ldq + (size_t)f.head * p.hd;
        const T* GO = (const T*)p.go + f.row * p.ldg + (size_t)f.head * p.hd;
        const T* O = (const T*)p.o + f.row * p.ldo + (size_t)f.head * p.hd;
        float dd = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int d = ks * M::KSTEP + (lane >> 5) * M::VEC;
            fq[g][ks] = fg[g][ks] = frag{};
            if (ok && d < p.hd) {
                fq[g][ks] = *reinterpret_cast<const frag*>(Q + d);
                fg[g][ks] = *reinterpret_cast<const frag*>(GO + d);
                const frag o = *reinterpret_cast<const frag*>(O + d);
#pragma unroll
                for (int j = 0; j < M::VEC; ++j) dd = fmaf((float)fg[g][ks][j], (float)o[j], dd);
            }
        }
        const float2 h = both_halves(dd);
        D[g] = h.x + h.y;
        float l = ok ? p.lse[((size_t)b * p.H + f.head) * p.nq + (f.row - (size_t)b * p.nq)] * LOG2E : 0.f;
        l2[g] = l == -INFINITY ? 0.f : l;   // an image that shows nothing: no tile below has a visible key
#pragma unroll
        for (int dg = 0; dg < DG; ++dg) zero16(dq[g][dg]);
    }
    const float c = p.c;
    const bool idle = (qt * 4 + wave) * 32 * QG >= p.R;

    // one walk over the block's keys: unit(buf, kb, s, dp) for every 32 of them, s hidden where it has to be
    auto walk = [&](auto unit) {
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
                    f32x16 s[QG], dp[QG];
#pragma unroll
                    for (int g = 0; g < QG; ++g) {
                        zero16(s[g]);
                        zero16(dp[g]);
                    }
                    const int off = (32 * kb + (lane & 31)) * L::STR + (lane >> 5) * L::VEC;
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        const frag kf = *reinterpret_cast<const frag*>(&sK[buf][off + ks * M::KSTEP]);
                        const frag vf = *reinterpret_cast<const frag*>(&sV[buf][off + ks * M::KSTEP]);
#pragma unroll
                        for (int g = 0; g < QG; ++g) {
                            M::rows(s[g], kf, fq[g][ks]);
                            M::rows(dp[g], vf, fg[g][ks]);
                        }
                    }
                    const auto hider = M::hider(!(((unsigned)(bits >> (32 * kb)) >> (lane & 31)) & 1), lane);
#pragma unroll
                    for (int g = 0; g < QG; ++g) M::hide(s[g], hider, lane);
                    unit(buf, kb, s, dp);
                }
            }
            if (more) {
                bits = __ballot(vis);
                store(buf ^ 1, bits);
            }
            __syncthreads();
        }
    };
    if constexpr (EXACT_D) {   // D = sum_k p dp in fp32, by a walk of its own
        float d0[QG], d1[QG];
#pragma unroll
        for (int g = 0; g < QG; ++g) d0[g] = d1[g] = 0.f;
        walk([&](int, int, const f32x16* s, const f32x16* dp) {
#pragma unroll
            for (int g = 0; g < QG; ++g)
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    d0[g] = fmaf(__builtin_amdgcn_exp2f(fmaf(s[g][r], c, -l2[g])), dp[g][r], d0[g]);
                    d1[g] = fmaf(__builtin_amdgcn_exp2f(fmaf(s[g][r + 1], c, -l2[g])), dp[g][r + 1], d1[g]);
                }
        });
#pragma unroll
        for (int g = 0; g < QG; ++g) {
            const float2 h = both_halves(d0[g] + d1[g]);
            D[g] = h.x + h.y;
        }
    }
#pragma unroll
    for (int g = 0; g < QG; ++g) {
        const int r = row0 + 32 * g;
        if (r < p.R && split == 0 && lane < 32) p.ld[(size_t)bk * p.R + r] = make_float2(l2[g], D[g]);
    }
    walk([&](int buf, int kb, const f32x16* s, const f32x16* dp) {
        typename M::Prob ds[QG];
#pragma unroll
        for (int g = 0; g < QG; ++g) {
            float v[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) v[r] = __builtin_amdgcn_exp2f(fmaf(s[g][r], c, -l2[g])) * (dp[g][r] - D[g]);
            ds[g] = M::pack(v);
        }
#pragma unroll
        for (int dg = 0; dg < DG; ++dg) {
            const auto kt = M::template col_frags<L::STR>(&sK[buf][32 * kb * L::STR + 32 * dg], lane);
#pragma unroll
            for (int g = 0; g < QG; ++g) M::cols(dq[g][dg], kt, ds[g]);
        }
    });
#pragma unroll
    for (int g = 0; g < QG; ++g) {
        const int r = row0 + 32 * g;
        if (r >= p.R) continue;
        const RowRef f = row_ref(p, b, kv, r);
        T* dst = (T*)p.dq + f.row * p.ld_dq + (size_t)f.head * p.hd;
        float* part = p.part_q + (((size_t)split * p.B * p.KV + bk) * p.R + r) * p.hd;
#pragma unroll
        for (int dg = 0; dg < DG; ++dg)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                float v[8];
                gather8(dq[g][dg], t, v);
                const int d = 32 * dg + 16 * t + 8 * (lane >> 5);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] *= p.scale;
                if (d < p.hd) {
                    if (p.qsplits > 1) store8(part + d, v);
                    else store8(dst + d, v);
                }
            }
    }
}

// ---------------------------------------------------------------------------------------- dk, dv
// Bound by vector issue too: four products a unit, P and dS rounded in between, lse and D of every row read from LDS.  The same case
// takes 147 us (410 TF of 10 hd flops a pair together with the rows kernel; 614 over images of one length).
// KW waves across the keys (32 each); the 4 / KW waves of one key group take the 32-row blocks of a tile in turn
template <typename T, int HD, int KW>
__global__ void __launch_bounds__(256) xattn_dkv_kernel(BArgs p) {
    typedef Tile<T, HD> L;
    typedef typename L::M M;
    typedef typename M::frag frag;
    constexpr int WR = 4 / KW, RT = 32 * (WR > 2 ? WR : 2), NC = RT * L::CPR / 256, KS = HD / M::KSTEP, DG = HD / 32;
    constexpr int TILE = RT * L::STR, JSTR = HD + 1;
    constexpr size_t LOOP = (size_t)4 * TILE * sizeof(T), JOIN = WR > 1 ? (size_t)4 * 32 * JSTR * 4 : 0;
    __shared__ __attribute__((aligned(16))) char smem[LOOP > JOIN ? LOOP : JOIN];
    __shared__ __attribute__((aligned(16))) float sL[2][RT], sD[2][RT];
    T* sQ = reinterpret_cast<T*>(smem);            // [2][TILE]
    T* sG = sQ + 2 * TILE;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, kw = wave % KW, wr = wave / KW;
    const unsigned vid = xcd_order(blockIdx.x, p.kblocks);
    const Item it = block_item(vid, p.KV, p.B, p.ksplits, p.ktiles, p.lens != nullptr);
    const int b = it.b, kv = it.kv, split = it.part, kt = it.tile, bk = b * p.KV + kv;
    int begin = 0, end = p.R;
    if (p.ksplits > 1) {
        const int tiles = (p.R + RT - 1) / RT, per = (tiles + p.ksplits - 1) / p.ksplits;
        begin = min(p.R, split * per * RT);
        end = min(p.R, (split + 1) * per * RT);
    }
    frag rq[NC], rg[NC];
    float2 rl;
    const int width = p.hd * (int)sizeof(T);
    const size_t ldqb = p.ldq * sizeof(T), ldgb = p.ldg * sizeof(T);
    const T* Q = (const T*)p.q + (size_t)b * p.nq * p.ldq + (size_t)kv * p.G * p.hd;
    const T* GO = (const T*)p.go + (size_t)b * p.nq * p.ldg + (size_t)kv * p.G * p.hd;
    // a tile's packed rows lie in the rows from the first one's query on, G heads side by side: a buffer at that query.  RT - 1 rows and
    // one row's heads stay below 2^31 bytes: 63 x 32 MB, or 127 x 16 MB by the launch rule of kw = 1
    auto load = [&](int r0) {
        const int q0 = (int)p.by_g.quot((unsigned)r0);
        const __amdgpu_buffer_rsrc_t qb = tile_buffer(Q, ldqb, q0, p.nq, width * p.G), gb = tile_buffer(GO, ldgb, q0, p.nq, width * p.G);
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int ci = tid + 256 * i, col = ci % L::CPR * 16, r = r0 + ci / L::CPR;
            const unsigned qi = p.by_g.quot((unsigned)r), in_row = (r - qi * p.G) * width + col;
            const bool ok = r < end && col < width;
            rq[i] = buffer_frag<frag>(qb, ok ? (qi - q0) * (unsigned)ldqb + in_row : 0x80000000u);
            rg[i] = buffer_frag<frag>(gb, ok ? (qi - q0) * (unsigned)ldgb + in_row : 0x80000000u);
        }
        rl = make_float2(0.f, 0.f);
        if (tid < RT && r0 + tid < end) rl = p.ld[(size_t)bk * p.R + r0 + tid];
    };
    auto store = [&](int buf) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int ci = tid + 256 * i, row = ci / L::CPR, d = (ci % L::CPR) * L::VEC;
            *reinterpret_cast<frag*>(&sQ[buf * TILE + row * L::STR + d]) = rq[i];
            *reinterpret_cast<frag*>(&sG[buf * TILE + row * L::STR + d]) = rg[i];
        }
        if (tid < RT) {
            sL[buf][tid] = rl.x;
            sD[buf][tid] = rl.y;
        }
    };
    // rows, keys and mask are asked for together: one latency, not three in a row
    if (begin < end) load(begin);
    const int key = kt * 32 * KW + 32 * kw + (lane & 31), krow = min(key, p.nk - 1);
    frag fk[KS], fv[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const int d = ks * M::KSTEP + (lane >> 5) * M::VEC;
        fk[ks] = fv[ks] = frag{};
        if (d < p.hd) {
            fk[ks] = *reinterpret_cast<const frag*>((const T*)p.k + ((size_t)b * p.nk + krow) * p.ldk + (size_t)kv * p.hd + d);
            fv[ks] = *reinterpret_cast<const frag*>((const T*)p.v + ((size_t)b * p.nk + krow) * p.ldv + (size_t)kv * p.hd + d);
        }
    }
    const bool shown = !p.mask || p.mask[(size_t)b * p.ldm + krow], vis = key < image_len(p, b) && shown;
    f32x16 dk[DG], dv[DG];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
        if (!vis) fk[ks] = fv[ks] = frag{};
#pragma unroll
    for (int dg = 0; dg < DG; ++dg) {
        zero16(dk[dg]);
        zero16(dv[dg]);
    }
    // a block whose keys are all hidden has nothing to add up
    if (!__syncthreads_or(vis)) end = begin;
    const bool idle = !__any(vis);

    const float c = p.c;
    if (begin < end) store(0);
    __syncthreads();
    int buf = 0;
    for (int r0 = begin; r0 < end; r0 += RT, buf ^= 1) {
        const bool more = r0 + RT < end;
        if (more) load(r0 + RT);
        if (!idle) {
#pragma unroll
            for (int i = 0; i < RT / 32 / WR; ++i) {
                const int rb = WR == 1 ? i : i * WR + wr;
                const T* tq = sQ + buf * TILE + 32 * rb * L::STR;
                const T* tg = sG + buf * TILE + 32 * rb * L::STR;
                const int off = (lane & 31) * L::STR + (lane >> 5) * L::VEC;
                f32x16 s, dp;
                zero16(s);
                zero16(dp);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    M::rows(s, *reinterpret_cast<const frag*>(tq + off + ks * M::KSTEP), fk[ks]);
                    M::rows(dp, *reinterpret_cast<const frag*>(tg + off + ks * M::KSTEP), fv[ks]);
                }
                float pr[16], ds[16];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const f32x4 l = *reinterpret_cast<const f32x4*>(&sL[buf][32 * rb + 8 * u + 4 * (lane >> 5)]);
                    const f32x4 D = *reinterpret_cast<const f32x4*>(&sD[buf][32 * rb + 8 * u + 4 * (lane >> 5)]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        // (a hidden key's lane holds anything: it is a column of its own to the end)
                        pr[4 * u + j] = __builtin_amdgcn_exp2f(fmaf(s[4 * u + j], c, -l[j]));
                        ds[4 * u + j] = pr[4 * u + j] * (dp[4 * u + j] - D[j]);
                    }
                }
                const typename M::Prob pp = M::pack(pr), pd = M::pack(ds);
#pragma unroll
                for (int dg = 0; dg < DG; ++dg) {
                    M::template cols<L::STR>(dv[dg], tg + 32 * dg, lane, pp);
                    M::template cols<L::STR>(dk[dg], tq + 32 * dg, lane, pd);
                }
            }
        }
        if (more) store(buf ^ 1);
        __syncthreads();
    }
    if constexpr (WR > 1) {   // join the row waves of each key group, dk first, then dv
        float* sj = reinterpret_cast<float*>(smem);
        auto join = [&](f32x16* a) {
#pragma unroll
            for (int dg = 0; dg < DG; ++dg)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    sj[(wave * 32 + (lane & 31)) * JSTR + 32 * dg + (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5)] = a[dg][r];
            __syncthreads();
#pragma unroll
            for (int dg = 0; dg < DG; ++dg)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float t = 0.f;
#pragma unroll
                    for (int w = 0; w < WR; ++w)
                        t += sj[((w * KW + kw) * 32 + (lane & 31)) * JSTR + 32 * dg + (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5)];
                    a[dg][r] = t;
                }
            __syncthreads();
        };
        join(dk);
        join(dv);
        if (wr != 0) return;
    }
    if (key >= p.nk) return;
    const size_t row = (size_t)b * p.nk + key;
    T* ok = (T*)p.dk + row * p.ld_dk + (size_t)kv * p.hd;
    T* ov = (T*)p.dv + row * p.ld_dv + (size_t)kv * p.hd;
    const size_t po = (((size_t)split * p.B * p.nk + row) * p.KV + kv) * p.hd;
#pragma unroll
    for (int dg = 0; dg < DG; ++dg)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            float a[8], v[8];
            gather8(dk[dg], t, a);
            gather8(dv[dg], t, v);
            const int d = 32 * dg + 16 * t + 8 * (lane >> 5);
#pragma unroll
            for (int j = 0; j < 8; ++j) a[j] = vis ? a[j] * p.scale : 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = vis ? v[j] : 0.f;
            if (d < p.hd) {
                if (p.ksplits > 1) {
                    store8(p.part_k + po + d, a);
                    store8(p.part_v + po + d, v);
                } else {
                    store8(ok + d, a);
                    store8(ov + d, v);
                }
            }
        }
}

// ---------------------------------------------------------------------------------------- few keys: all three at once
// Up to 32 NKB keys (captions, ViT states): K and V of a key head stay in LDS, its dk and dv in registers, and every row of q
// and dout is read once.  Per unit (32 rows x 32 keys): S^T = K q^T and dP^T = V dout^T from LDS and registers, dq^T += K^T dS
// from registers; P and dS go through a patch of LDS of the wave's own and come back transposed for dv^T += dout^T P and
// dk^T += q^T dS.  5 products instead of 7.  The four waves' dk, dv (and the parts over blocks) are summed in order at the end.
// Against the two kernels below it: 8 x 64 x 64 queries over 77 states, 8 heads of 32, 53 -> 33 us; over 50, 8 heads of 64, 66 -> 47 us.
template <int HD, int NKB>
__global__ void __launch_bounds__(256, 2) xattn_short_bwd_kernel(BArgs p) {
    typedef bf16_t T;
    typedef Tile<T, HD> L;
    typedef Mma<T> M;
    typedef M::frag frag;
    constexpr int KS = HD / 16, DG = HD / 32, STR = L::STR, PSTR = 32 + M::PAD, JSTR = HD + 4;
    constexpr int KVT = NKB * 32 * STR, WT = 2 * 32 * STR + 2 * 32 * PSTR;   // elements: K (or V), a wave's patch
    constexpr int LOOP = (2 * KVT + 4 * WT) * 2, JOIN = 2 * 4 * 32 * JSTR * 4;
    constexpr bool AHEAD = NKB * DG < 4;   // registers left to fetch the next rows while these are worked on
    __shared__ __attribute__((aligned(16))) char smem[LOOP > JOIN ? LOOP : JOIN];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    T* sK = reinterpret_cast<T*>(smem);
    T* sV = sK + KVT;
    T* sQ = sV + KVT + wave * WT;
    T* sG = sQ + 32 * STR;
    T* sP = sG + 32 * STR;
    T* sS = sP + 32 * PSTR;
    const unsigned vid = xcd_order(blockIdx.x, p.kblocks);
    const Item it = block_item(vid, p.KV, p.B, p.ksplits, 1, p.lens != nullptr);
    const int b = it.b, kv = it.kv, split = it.part, row = lane & 31, half = lane >> 5;
    const int steps = (p.R + 127) / 128, per = (steps + p.ksplits - 1) / p.ksplits;
    const int begin = min(p.R, split * per * 128), end = min(p.R, (split + 1) * per * 128);

    frag fq[KS], fg[KS];
    float l2 = 0.f;
    auto fetch = [&](int r) {   // row r of q, dout and its lse; zeros behind the last row
        const bool ok = r < end;
        const RowRef f = row_ref(p, b, kv, ok ? r : 0);
        const T* Q = (const T*)p.q + f.row * p.ldq + (size_t)f.head * p.hd;
        const T* GO = (const T*)p.go + f.row * p.ldg + (size_t)f.head * p.hd;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int d = ks * 16 + half * 8;
            fq[ks] = fg[ks] = frag{};
            if (ok && d < p.hd) {
                fq[ks] = *reinterpret_cast<const frag*>(Q + d);
                fg[ks] = *reinterpret_cast<const frag*>(GO + d);
            }
        }
        l2 = ok ? p.lse[((size_t)b * p.H + f.head) * p.nq + (f.row - (size_t)b * p.nq)] : 0.f;
    };
    int r0 = begin + wave * 32;
    if (AHEAD && r0 < end) fetch(r0 + row);
    // ---- keys of the whole image
    const int len = image_len(p, b);
    const unsigned char* mask = p.mask ? p.mask + (size_t)b * p.ldm : nullptr;
    {
        const T* K = (const T*)p.k + (size_t)b * p.nk * p.ldk + (size_t)kv * p.hd;
        const T* V = (const T*)p.v + (size_t)b * p.nk * p.ldv + (size_t)kv * p.hd;
        for (int i = tid; i < NKB * 32 * L::CPR; i += 256) {
            const int key = i / L::CPR, d = i % L::CPR * 8;
            frag a = frag{}, c = frag{};
            if (key < len && d < p.hd && (!mask || mask[key])) {
                a = *reinterpret_cast<const frag*>(K + (size_t)key * p.ldk + d);
                c = *reinterpret_cast<const frag*>(V + (size_t)key * p.ldv + d);
            }
            *reinterpret_cast<frag*>(sK + key * STR + d) = a;
            *reinterpret_cast<frag*>(sV + key * STR + d) = c;
        }
    }
    unsigned hidden = 0;   // bit kb: this lane's key of block kb
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb) {
        const int key = 32 * kb + row;
        if (!(key < len && (!mask || mask[key]))) hidden |= 1u << kb;
    }
    __syncthreads();

    f32x16 dk[NKB][DG], dv[NKB][DG];
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
        for (int dg = 0; dg < DG; ++dg) {
            zero16(dk[kb][dg]);
            zero16(dv[kb][dg]);
        }
    const float c = p.c;
    for (; r0 < end; r0 += 128) {
        // ---- this group's rows: q and dout into the wave's patch
        if (!AHEAD) fetch(r0 + row);
        const float lr = l2 == -INFINITY ? 0.f : l2 * LOG2E;
        frag q[KS], g[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            q[ks] = fq[ks];
            g[ks] = fg[ks];
            *reinterpret_cast<frag*>(sQ + row * STR + ks * 16 + half * 8) = q[ks];
            *reinterpret_cast<frag*>(sG + row * STR + ks * 16 + half * 8) = g[ks];
        }
        if (AHEAD && r0 + 128 < end) fetch(r0 + 128 + row);
        auto products = [&](int kb, f32x16& s, f32x16& dp) {
            zero16(s);
            zero16(dp);
            const int off = (32 * kb + row) * STR + half * 8;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                M::rows(s, *reinterpret_cast<const frag*>(sK + off + ks * 16), q[ks]);
                M::rows(dp, *reinterpret_cast<const frag*>(sV + off + ks * 16), g[ks]);
            }
            M::hide(s, M::hider((hidden >> kb) & 1, lane), lane);
        };
        // D = sum_k p dp of the row in fp32, with all keys at hand.  dout . out would be one product, but out is rounded: over few
        // keys that alone moved dq and dk by 0.001 of their norm, next to 0.0017 for their own rounding.
        float D0 = 0.f, D1 = 0.f;
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) {
            f32x16 s, dp;
            products(kb, s, dp);
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                D0 = fmaf(__builtin_amdgcn_exp2f(fmaf(s[r], c, -lr)), dp[r], D0);
                D1 = fmaf(__builtin_amdgcn_exp2f(fmaf(s[r + 1], c, -lr)), dp[r + 1], D1);
            }
        }
        const float2 hs = both_halves(D0 + D1);
        const float D = hs.x + hs.y;
        f32x16 dq[DG];
#pragma unroll
        for (int dg = 0; dg < DG; ++dg) zero16(dq[dg]);
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) {
            f32x16 s, dp;
            products(kb, s, dp);
            float pr[16], ds[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                pr[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -lr));
                ds[r] = pr[r] * (dp[r] - D);
            }
            const M::Prob pp = M::pack(pr), pd = M::pack(ds);
#pragma unroll
            for (int dg = 0; dg < DG; ++dg) M::cols<STR>(dq[dg], sK + 32 * kb * STR + 32 * dg, lane, pd);
#pragma unroll
            for (int u = 0; u < 4; ++u) {   // quad u of the registers: keys 8 u + 4 half + 0..3 of this lane's row
                bf16x4 a, e;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    a[j] = pp.p[u >> 1][4 * (u & 1) + j];
                    e[j] = pd.p[u >> 1][4 * (u & 1) + j];
                }
                *reinterpret_cast<bf16x4*>(sP + row * PSTR + 8 * u + 4 * half) = a;
                *reinterpret_cast<bf16x4*>(sS + row * PSTR + 8 * u + 4 * half) = e;
            }
            // the wave's own LDS operations stay in order; only the compiler has to be held
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            const M::ColFrags pf = M::col_frags<PSTR>(sP, lane), sf = M::col_frags<PSTR>(sS, lane);
#pragma unroll
            for (int dg = 0; dg < DG; ++dg) {
                const M::ColFrags gf = M::col_frags<STR>(sG + 32 * dg, lane), qf = M::col_frags<STR>(sQ + 32 * dg, lane);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    dv[kb][dg] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(gf.f[t], pf.f[t], dv[kb][dg], 0, 0, 0);
                    dk[kb][dg] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qf.f[t], sf.f[t], dk[kb][dg], 0, 0, 0);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
        const int r = r0 + row;
        if (r < end) {
            const RowRef f = row_ref(p, b, kv, r);
            T* dst = (T*)p.dq + f.row * p.ld_dq + (size_t)f.head * p.hd;
#pragma unroll
            for (int dg = 0; dg < DG; ++dg)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    float v[8];
                    gather8(dq[dg], t, v);
                    const int d = 32 * dg + 16 * t + 8 * half;
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] *= p.scale;
                    if (d < p.hd) store8(dst + d, v);
                }
        }
    }
    // ---- the four waves' sums, one 32-key block at a time: dk and dv side by side
    float* sj = reinterpret_cast<float*>(smem);
    constexpr int ONE = 4 * 32 * JSTR;
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb) {
        __syncthreads();
#pragma unroll
        for (int dg = 0; dg < DG; ++dg)
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                f32x4 v, w;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[j] = dk[kb][dg][4 * u + j];
                    w[j] = dv[kb][dg][4 * u + j];
                }
                float* at = sj + (wave * 32 + row) * JSTR + 32 * dg + 8 * u + 4 * half;
                *reinterpret_cast<f32x4*>(at) = v;
                *reinterpret_cast<f32x4*>(at + ONE) = w;
            }
        __syncthreads();
        for (int i = tid; i < 2 * 32 * (HD / 8); i += 256) {
            const int which = i / (32 * (HD / 8)), k32 = i / (HD / 8) % 32, d = i % (HD / 8) * 8, key = 32 * kb + k32;
            if (key >= p.nk || d >= p.hd) continue;
            const bool vis = key < len && (!mask || mask[key]);
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w)
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] += sj[which * ONE + (w * 32 + k32) * JSTR + d + j];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = vis ? (which ? v[j] : v[j] * p.scale) : 0.f;
            const size_t krow = (size_t)b * p.nk + key;
            if (p.ksplits > 1)
                store8((which ? p.part_v : p.part_k) + (((size_t)split * p.B * p.nk + krow) * p.KV + kv) * p.hd + d, v);
            else
                store8((which ? (T*)p.dv + krow * p.ld_dv : (T*)p.dk + krow * p.ld_dk) + (size_t)kv * p.hd + d, v);
        }
    }
}

// out[row][d] = sum over the parts, in order; one thread per row, head and 8 columns.  grid.y: 0 = dk, 1 = dv
template <typename T>
__global__ void __launch_bounds__(256) xattn_sum_keys_kernel(BArgs p) {
    const int cpr = p.KV * p.hd / 8;
    const size_t rows = (size_t)p.B * p.nk, i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= rows * cpr) return;
    const size_t row = i / cpr, d = 8 * (i % cpr), stride = rows * p.KV * p.hd;
    const float* src = (blockIdx.y ? p.part_v : p.part_k) + row * p.KV * p.hd + d;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
#pragma unroll 8
    for (int s = 0; s < p.ksplits; ++s) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(src + s * stride), e = *reinterpret_cast<const f32x4*>(src + s * stride + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] += a[j];
            v[4 + j] += e[j];
        }
    }
    store8(blockIdx.y ? (T*)p.dv + row * p.ld_dv + d : (T*)p.dk + row * p.ld_dk + d, v);
}

template <typename T>
__global__ void __launch_bounds__(256) xattn_sum_rows_kernel(BArgs p) {
    const int cpr = p.hd / 8;
    const size_t rows = (size_t)p.B * p.KV * p.R, i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= rows * cpr) return;
    const size_t pr = i / cpr;
    const int d = 8 * (int)(i % cpr);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
#pragma unroll 8
    for (int s = 0; s < p.qsplits; ++s) {
        const float* src = p.part_q + (s * rows + pr) * p.hd + d;
        const f32x4 a = *reinterpret_cast<const f32x4*>(src), e = *reinterpret_cast<const f32x4*>(src + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] += a[j];
            v[4 + j] += e[j];
        }
    }
    const int r = (int)(pr % p.R), kv = (int)(pr / p.R % p.KV), b = (int)(pr / p.R / p.KV);
    const RowRef f = row_ref(p, b, kv, r);
    store8((T*)p.dq + f.row * p.ld_dq + (size_t)f.head * p.hd + d, v);
}

// ---------------------------------------------------------------------------------------- launch rules
struct Plan {
    int few;    // blocks of 32 keys of the one-kernel form, 0: two kernels
    bool exact; // dq: D by a walk of its own
    bool two;   // dq: two row groups a wave
    int qsplits, qtiles, kw, ksplits, ktiles;
};

// parts of an axis of `tiles` steps so that `blocks` blocks grow to about two per CU, each with two steps at least
int parts(long long blocks, long long tiles) {
    long long s = blocks >= 384 ? 1 : (512 + blocks - 1) / (blocks > 0 ? blocks : 1);
    if (s > tiles / 2) s = tiles / 2;
    if (s > 64) s = 64;
    return s < 1 ? 1 : (int)s;
}

// `far`: rows of q or dout lie 16 MB apart or more
Plan plan_bwd(int B, int nq, int nk, int H, int KV, int hd, int dtype, bool ragged, bool far) {
    Plan pl = {};
    const long long R = (long long)nq * (H / KV), bk = (long long)B * KV, wide = (R + 255) / 256 * bk;
    // one kernel where dk and dv of all keys fit a wave's registers
    if (dtype == UWIR_BF16 && nq > 0 && nk > 0 && hd <= 64 && nk <= (hd <= 32 ? 128 : 64)) {
        pl.few = (nk + 31) / 32;
        pl.qsplits = 1;
        pl.ksplits = parts(bk, (R + 127) / 128);
        return pl;
    }
    pl.exact = dtype == UWIR_BF16 && nk <= 256;
    pl.qsplits = pl.exact ? 1 : parts(bk * ((R + 127) / 128), (nk + 63) / 64);
    // 256 rows a block (bf16, up to 64 columns) where two such blocks a CU remain; with lengths per image, where the longest image's
    // blocks set the time, only from eight on.  4 x 64 x 64 queries over 2048 states, 8 heads of 64: 273 against 310 us; ragged and
    // with shared heads 248 against 241.
    pl.two = dtype == UWIR_BF16 && !pl.exact && hd <= 64 && R > 128 && pl.qsplits == 1 && wide >= (ragged ? 2048 : 512);
    pl.qtiles = (int)((R + (pl.two ? 255 : 127)) / (pl.two ? 256 : 128));
    // few keys: waves beyond them take rows instead (fp32 rows of 128 columns leave no LDS for the longer row tiles; the 128 rows of
    // kw = 1 have to lie within the 2^31 bytes of a buffer, those of kw = 2 are 64.  Both have the same parts for 32 keys)
    pl.kw = hd > 64 && dtype == UWIR_F32 ? 4 : nk <= 32 && !far ? 1 : nk <= 64 ? 2 : 4;
    pl.ktiles = (nk + 32 * pl.kw - 1) / (32 * pl.kw);
    pl.ksplits = parts(bk * pl.ktiles, (R + 63) / 64);
    return pl;
}

struct Layout {
    size_t ld, q, k, v, total;
};
Layout layout(const Plan& pl, int B, int nq, int nk, int H, int KV, int hd) {
    Layout l;
    size_t at = al256((size_t)B * H * nq * sizeof(float2));
    l.ld = 0;
    l.q = at;
    if (pl.qsplits > 1) at += al256((size_t)pl.qsplits * B * H * nq * hd * 4);
    l.k = at;
    if (pl.ksplits > 1) at += al256((size_t)pl.ksplits * B * nk * KV * hd * 4);
    l.v = at;
    if (pl.ksplits > 1) at += al256((size_t)pl.ksplits * B * nk * KV * hd * 4);
    l.total = at;
    return l;
}

template <typename T> void launch_sum_keys(const BArgs& p, hipStream_t st) {
    if (p.ksplits == 1) return;
    const size_t n = (size_t)p.B * p.nk * p.KV * (p.hd / 8);
    hipLaunchKernelGGL((xattn_sum_keys_kernel<T>), dim3((unsigned)ceil_div_sz(n, 256), 2), dim3(256), 0, st, p);
}

template <typename T, int HD> void launch(const BArgs& p, const Plan& pl, hipStream_t st) {
    if constexpr (sizeof(T) == 2 && HD <= 64) {
        if (pl.few) {
            const dim3 grid(p.kblocks), block(256);
            if (pl.few == 1) hipLaunchKernelGGL((xattn_short_bwd_kernel<HD, 1>), grid, block, 0, st, p);
            if (pl.few == 2) hipLaunchKernelGGL((xattn_short_bwd_kernel<HD, 2>), grid, block, 0, st, p);
            if constexpr (HD == 32) {
                if (pl.few == 3) hipLaunchKernelGGL((xattn_short_bwd_kernel<HD, 3>), grid, block, 0, st, p);
                if (pl.few == 4) hipLaunchKernelGGL((xattn_short_bwd_kernel<HD, 4>), grid, block, 0, st, p);
            }
            launch_sum_keys<T>(p, st);
            return;
        }
    }
    if (p.nq > 0) {
        const dim3 grid(p.qblocks), block(256);
        bool done = false;
        if constexpr (sizeof(T) == 2) {
            if (pl.exact) {
                hipLaunchKernelGGL((xattn_dq_kernel<T, HD, 1, true>), grid, block, 0, st, p);
                done = true;
            } else if constexpr (HD <= 64) {
                if (pl.two) {
                    hipLaunchKernelGGL((xattn_dq_kernel<T, HD, 2, false>), grid, block, 0, st, p);
                    done = true;
                }
            }
        }
        if (!done) hipLaunchKernelGGL((xattn_dq_kernel<T, HD, 1, false>), grid, block, 0, st, p);
        if (p.qsplits > 1) {
            const size_t n = (size_t)p.B * p.KV * p.R * (p.hd / 8);
            hipLaunchKernelGGL((xattn_sum_rows_kernel<T>), dim3((unsigned)ceil_div_sz(n, 256)), dim3(256), 0, st, p);
        }
    }
    if (p.nk > 0) {
        if constexpr (sizeof(T) == 2 || HD <= 64) {
            if (pl.kw == 1) hipLaunchKernelGGL((xattn_dkv_kernel<T, HD, 1>), dim3(p.kblocks), dim3(256), 0, st, p);
            if (pl.kw == 2) hipLaunchKernelGGL((xattn_dkv_kernel<T, HD, 2>), dim3(p.kblocks), dim3(256), 0, st, p);
        }
        if (pl.kw == 4) hipLaunchKernelGGL((xattn_dkv_kernel<T, HD, 4>), dim3(p.kblocks), dim3(256), 0, st, p);
        launch_sum_keys<T>(p, st);
    }
}

}  // namespace

extern "C" size_t uwir_cross_attn_backward_workspace_bytes(int B, int nq, int nk, int heads, int kv_heads, int hd, int dtype) {
    if (B <= 0 || nq < 0 || nk < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || hd <= 0) return 0;
    return layout(plan_bwd(B, nq, nk, heads, kv_heads, hd, dtype, false, false), B,   // the parts do not depend on lengths and strides
                   nq, nk, heads, kv_heads, hd).total;
}

extern "C" int uwir_cross_attn_backward(const void* q, size_t ldq, const void* k, size_t ldk, const void* v, size_t ldv,
                                        const void* out, size_t ldo, const float* lse, const void* dout, size_t ld_dout, int dtype,
                                        int B, int nq, int nk, int heads, int kv_heads, int hd, float scale, const int* key_lens,
                                        const unsigned char* key_mask, size_t ld_mask, void* dq, size_t ld_dq, void* dk,
                                        size_t ld_dk, void* dv, size_t ld_dv, void* workspace, size_t workspace_bytes,
                                        uwir_stream_t stream) {
    if (int rc = xattn_check("cross_attn_backward", dtype, B, nq, nk, heads, kv_heads, hd, scale)) return rc;
    if (nq == 0 && nk == 0) return UWIR_OK;
    const size_t rq = (size_t)B * nq, rk = (size_t)B * nk;
    const XMat in[] = {{q, ldq, heads, rq, "q"}, {k, ldk, kv_heads, rk, "k"}, {v, ldv, kv_heads, rk, "v"}, {out, ldo, heads, rq, "out"},
                       {dout, ld_dout, heads, rq, "dout"}};
    const XMat res[] = {{dq, ld_dq, heads, rq, "dq"}, {dk, ld_dk, kv_heads, rk, "dk"}, {dv, ld_dv, kv_heads, rk, "dv"}};
    if (int rc = xattn_check_mats("cross_attn_backward", dtype, hd, in, 5, res, 3)) return rc;
    UWIR_CHECK(nq == 0 || lse, "cross_attn_backward: null pointer (lse)");
    UWIR_CHECK(!key_mask || ld_mask >= (size_t)nk, "cross_attn_backward: mask rows must have at least nk entries");
    const size_t need = uwir_cross_attn_backward_workspace_bytes(B, nq, nk, heads, kv_heads, hd, dtype);
    UWIR_CHECK(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
               "cross_attn_backward: workspace too small or not 16-byte aligned");
    if (int rc = xattn_check_apart("cross_attn_backward", "the workspace", workspace, need, dtype, hd, in, 5)) return rc;
    if (int rc = xattn_check_apart("cross_attn_backward", "the workspace", workspace, need, dtype, hd, res, 3)) return rc;
    if (int rc = xattn_check_apart("cross_attn_backward", "lse", lse, (size_t)B * heads * nq * sizeof(float), dtype, hd, res, 3)) return rc;
    const uintptr_t w = (uintptr_t)workspace, ls = (uintptr_t)lse;
    UWIR_CHECK(!nq || w + need <= ls || ls + (size_t)B * heads * nq * sizeof(float) <= w, "cross_attn_backward: the workspace overlaps lse");
    const XRange beside[] = {{workspace, need, "the workspace"}};
    if (int rc = xattn_check_keys("cross_attn_backward", key_lens, key_mask, ld_mask, B, nk, dtype, hd, res, 3, beside, 1)) return rc;
    const size_t apart = (ldq > ld_dout ? ldq : ld_dout) * (dtype == UWIR_BF16 ? 2 : 4);
    const Plan pl = plan_bwd(B, nq, nk, heads, kv_heads, hd, dtype, key_lens != nullptr, apart >= (1u << 24));
    const Layout lo = layout(pl, B, nq, nk, heads, kv_heads, hd);
    BArgs p = {};
    p.q = q; p.k = k; p.v = v; p.o = out; p.go = dout; p.lse = lse; p.dq = dq; p.dk = dk; p.dv = dv;
    p.lens = key_lens; p.mask = key_mask;
    p.ldq = ldq; p.ldk = ldk; p.ldv = ldv; p.ldo = ldo; p.ldg = ld_dout; p.ld_dq = ld_dq; p.ld_dk = ld_dk; p.ld_dv = ld_dv;
    p.ldm = ld_mask;
    p.B = B; p.nq = nq; p.nk = nk; p.H = heads; p.KV = kv_heads; p.hd = hd; p.G = heads / kv_heads; p.R = nq * p.G;
    p.qsplits = pl.qsplits; p.qtiles = pl.qtiles; p.ksplits = pl.ksplits; p.ktiles = pl.ktiles;
    const long long qb = (long long)B * kv_heads * pl.qtiles * pl.qsplits, kb = (long long)B * kv_heads * (pl.few ? 1 : pl.ktiles) * pl.ksplits;
    UWIR_CHECK(qb < (1ll << 24) && kb < (1ll << 24), "cross_attn_backward: too many rows for one launch");   // 2^32 threads
    p.qblocks = (int)qb; p.kblocks = (int)kb;
    p.c = scale * LOG2E; p.scale = scale; p.by_g = make_divisor(p.G);
    char* ws = (char*)workspace;
    p.ld = (float2*)(ws + lo.ld);
    p.part_q = (float*)(ws + lo.q); p.part_k = (float*)(ws + lo.k); p.part_v = (float*)(ws + lo.v);
    hipStream_t st = (hipStream_t)stream;
    switch (hd_class(hd) + (dtype == UWIR_BF16)) {
        case 32: launch<float, 32>(p, pl, st); break;
        case 33: launch<bf16_t, 32>(p, pl, st); break;
        case 64: launch<float, 64>(p, pl, st); break;
        case 65: launch<bf16_t, 64>(p, pl, st); break;
        case 128: launch<float, 128>(p, pl, st); break;
        default: launch<bf16_t, 128>(p, pl, st); break;
    }
    UWIR_LAUNCH_CHECK("cross_attn_backward");
    return UWIR_OK;
}
