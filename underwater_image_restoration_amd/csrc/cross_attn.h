// Shared pieces of the cross-attention kernels (forward and backward).
//
// Everything is built on 32 x 32 accumulators of v_mfma_f32_32x32x16_bf16 / v_mfma_f32_32x32x2_f32, in which lane l holds
// column l % 32 and rows (r & 3) + 8 (r >> 2) + 4 (l / 32), r = 0..15.  A product whose summed index lies on the rows of
// such an accumulator takes it as its B operand straight from registers, as long as the A operand follows the same order
// of the summed index; so probabilities and score gradients never pass through shared memory.  The two A operands:
//   rows   row l % 32 of a row-major tile, 16 consecutive bytes a lane (K in K q^T, q in q K^T, ...)
//   cols   column l % 32 of the same tile, summed rows in accumulator order (V^T P, K^T dS, q^T dS, dO^T P): one
//          transposing LDS read per four rows (bf16), or plain reads (fp32, consecutive lanes = consecutive columns)
#pragma once
#include "common.h"

namespace xattn {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.69314718055994531f;

template <typename T> struct Mma;

template <> struct Mma<bf16_t> {
    static constexpr int VEC = 8, KSTEP = 16, PAD = 8;   // elements: per 16 bytes, per rows() step, of LDS row padding
    typedef bf16x8 frag;
    struct Prob { bf16x8 p[2]; };
    static __device__ __forceinline__ void rows(f32x16& acc, frag a, frag b) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0);
    }
    static __device__ __forceinline__ Prob pack(const float* v) {
        Prob o;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) o.p[s][j] = (bf16_t)v[8 * s + j];
        return o;
    }
    // Hides keys: one more step of rows() in which a hidden key's row carries the type's lowest value and every query a one, so
    // that its score is about -3.4e38 and its probability 0.  No select per score, no branch, one MFMA of a dozen.
    static __device__ __forceinline__ frag hider(bool hidden, int lane) {
        frag f;
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = (bf16_t)0.f;
        f[0] = lane < 32 && hidden ? __builtin_bit_cast(bf16_t, (unsigned short)0xff7f) : (bf16_t)0.f;
        return f;
    }
    static __device__ __forceinline__ void hide(f32x16& acc, frag hider, int lane) {
        frag one;
#pragma unroll
        for (int j = 0; j < 8; ++j) one[j] = (bf16_t)(j == 0 ? 1.f : 0.f);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(hider, one, acc, 0, 0, 0);
    }
    // acc[col0 + ., .] += tile[row0 .. row0 + 31][col0 + .]^T * prob.  Lane group of 16: four rows x 16 columns a read.
    struct ColFrags { frag f[2]; };
    template <int STR> static __device__ __forceinline__ ColFrags col_frags(const bf16_t* tile, int lane) {
        typedef __attribute__((address_space(3))) bf16x4 lds4;
        const bf16_t* p = tile + (4 * (lane >> 5) + ((lane & 15) >> 2)) * STR + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        ColFrags c;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4*)(p + 16 * s * STR));
            const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4*)(p + (16 * s + 8) * STR));
            c.f[s] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        return c;
    }
    static __device__ __forceinline__ void cols(f32x16& acc, const ColFrags& a, const Prob& b) {
#pragma unroll
        for (int s = 0; s < 2; ++s) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.f[s], b.p[s], acc, 0, 0, 0);
    }
    template <int STR> static __device__ __forceinline__ void cols(f32x16& acc, const bf16_t* tile, int lane, const Prob& b) {
        cols(acc, col_frags<STR>(tile, lane), b);
    }
};

template <> struct Mma<float> {
    static constexpr int VEC = 4, KSTEP = 8, PAD = 4;
    typedef f32x4 frag;
    struct Prob { float p[16]; };
    static __device__ __forceinline__ void rows(f32x16& acc, frag a, frag b) {
#pragma unroll
        for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], acc, 0, 0, 0);
    }
    static __device__ __forceinline__ Prob pack(const float* v) {
        Prob o;
#pragma unroll
        for (int r = 0; r < 16; ++r) o.p[r] = v[r];
        return o;
    }
    static __device__ __forceinline__ float hider(bool hidden, int lane) { return lane < 32 && hidden ? -3.38e38f : 0.f; }
    static __device__ __forceinline__ void hide(f32x16& acc, float hider, int lane) {
        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(hider, 1.f, acc, 0, 0, 0);
    }
    struct ColFrags { float f[16]; };
    template <int STR> static __device__ __forceinline__ ColFrags col_frags(const float* tile, int lane) {
        const float* p = tile + 4 * (lane >> 5) * STR + (lane & 31);
        ColFrags c;
#pragma unroll
        for (int r = 0; r < 16; ++r) c.f[r] = p[((r & 3) + 8 * (r >> 2)) * STR];
        return c;
    }
    static __device__ __forceinline__ void cols(f32x16& acc, const ColFrags& a, const Prob& b) {
#pragma unroll
        for (int r = 0; r < 16; ++r) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.f[r], b.p[r], acc, 0, 0, 0);
    }
    template <int STR> static __device__ __forceinline__ void cols(f32x16& acc, const float* tile, int lane, const Prob& b) {
        cols(acc, col_frags<STR>(tile, lane), b);
    }
};

__device__ __forceinline__ void zero16(f32x16& a) {
#pragma unroll
    for (int r = 0; r < 16; ++r) a[r] = 0.f;
}

// A tile of rows of a matrix in global memory as a buffer: rows from `row` on, of which those below `end` exist; anything
// beyond reads as zeros, so that neither clamps nor selects sit in the loops.  `ldb`, `width` in bytes, width <= ldb; a buffer holds
// 2^31 - 1 bytes: the rows that a block reaches in it times ldb stay below that (64 rows of ldb < 2^25).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_buffer(const void* base, size_t ldb, int row, int end, int width) {
    const size_t bytes = row < end ? (size_t)(end - row - 1) * ldb + width : 0;
    return __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)base + (size_t)row * ldb), 0,
                                             (int)(bytes < 0x7fffffff ? bytes : 0x7fffffff), 0x00020000);
}
// byte offset of a 16-byte chunk in such a buffer; columns behind the matrix lie behind every buffer
__device__ __forceinline__ unsigned tile_offset(int row, unsigned ldb, int col_bytes, int width) {
    return col_bytes < width ? row * ldb + col_bytes : 0x80000000u;
}
template <typename F> __device__ __forceinline__ F buffer_frag(__amdgpu_buffer_rsrc_t r, unsigned off) {
    return __builtin_bit_cast(F, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0));
}

// v of this lane and of lane ^ 32, in an order that depends on the half: for symmetric uses
__device__ __forceinline__ float2 both_halves(float v) {
    const unsigned u = __float_as_uint(v);
    auto sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return make_float2(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
}

// Accumulator rows 8q .. 8q+7 of a 32-row block (q = 0..3) sit as two quads, one in each half of the wave.  Swapping
// quads between the halves leaves every lane with 8 consecutive rows: rows 16 t + 8 half + 0..7 for t = 0, 1.
__device__ __forceinline__ void gather8(const f32x16& a, int t, float* o) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(a[8 * t + j]), __float_as_uint(a[8 * t + 4 + j]), false, false);
        o[j] = __uint_as_float(sw[0]);
        o[4 + j] = __uint_as_float(sw[1]);
    }
}

__device__ __forceinline__ void store8(bf16_t* p, const float* v) {
    bf16x8 o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = (bf16_t)v[j];
    *reinterpret_cast<bf16x8*>(p) = o;
}
__device__ __forceinline__ void store8(float* p, const float* v) {
    f32x4 a, b;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        a[j] = v[j];
        b[j] = v[4 + j];
    }
    *reinterpret_cast<f32x4*>(p) = a;
    *reinterpret_cast<f32x4*>(p + 4) = b;
}

// contiguous ranges of work per XCD (blocks are dealt to the 8 XCDs in turn): blocks that read the same keys share an L2
__device__ __forceinline__ unsigned xcd_order(unsigned bid, unsigned nblocks) {
    const unsigned q = nblocks / 8, r = nblocks % 8, x = bid % 8;
    return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + bid / 8;
}

// r / G for 0 <= r < 2^30 by one high product: G in (2^(sh - 1), 2^sh], mul = floor(2^32 (2^sh - G) / G) + 1
struct Divisor {
    unsigned mul, sh, d;
    __device__ __forceinline__ unsigned quot(unsigned r) const { return (__umulhi(r, mul) + r) >> sh; }
};
inline Divisor make_divisor(unsigned d) {
    Divisor v = {0, 0, d};
    while ((1u << v.sh) < d) ++v.sh;
    v.mul = (unsigned)(((((unsigned long long)1 << v.sh) - d) << 32) / d + 1);
    return v;
}

template <typename T, int HD> struct Tile {
    typedef Mma<T> M;
    static constexpr int VEC = M::VEC, STR = HD + M::PAD, CPR = HD / VEC;   // 16-byte chunks per row
};

// the row of q / out that packed row r of key head kv stands for; Args: B, nq, G and by_g of either direction
struct RowRef {
    size_t row;
    int head;
};
template <typename Args> __device__ __forceinline__ RowRef row_ref(const Args& p, int b, int kv, int r) {
    const int qi = (int)p.by_g.quot((unsigned)r);
    return {(size_t)b * p.nq + qi, kv * p.G + (r - qi * p.G)};
}

// Which (head, image, part, tile) a block works on.  Heads next to each other: the blocks that run together read whole rows.
// Then, an XCD taking a contiguous range of the order: with all images of one length the images far apart, so that an XCD holds
// few images' keys in its L2; with lengths of their own next to each other, so that every XCD gets its share of the long ones.
struct Item {
    int kv, b, part, tile;
};
__device__ __forceinline__ Item block_item(unsigned vid, int KV, int B, int parts, int tiles, bool ragged) {
    Item it;
    it.kv = vid % KV;
    vid /= KV;
    if (ragged) {
        // turned by one image per round, and by one more per round of rounds: blocks go to the CUs in turn, and a CU that met
        // the same image every time would be done early or late
        unsigned turn = 0;
        if (B > 1)
            for (unsigned t = vid / B; t; t /= B) turn += t;
        it.b = (vid + turn) % B;
        vid /= B;
    }
    it.tile = vid % tiles;
    vid /= tiles;
    it.part = vid % parts;
    if (!ragged) it.b = vid / parts;
    return it;
}

}  // namespace xattn

// ---- host side: sizes and argument checks shared by both directions
namespace {

inline int hd_class(int hd) { return hd <= 32 ? 32 : hd <= 64 ? 64 : 128; }
inline size_t al256(size_t v) { return (v + 255) & ~(size_t)255; }

struct XMat {
    const void* p;
    size_t ld;
    int heads;
    size_t rows;
    const char* name;
};

inline int xattn_check(const char* what, int dtype, int B, int nq, int nk, int heads, int kv_heads, int hd, float scale) {
    UWIR_CHECK(dtype == UWIR_F32 || dtype == UWIR_BF16, "%s: bad dtype", what);
    UWIR_CHECK(B > 0 && nq >= 0 && nk >= 0, "%s: bad shape (B > 0, nq >= 0, nk >= 0)", what);
    UWIR_CHECK(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, "%s: kv_heads must divide heads", what);
    UWIR_CHECK((long long)B * kv_heads <= 65535 && (long long)nq * (heads / kv_heads) < (1ll << 30) && nk < (1 << 30),
               "%s: too large (B * kv_heads <= 65535; nq * heads / kv_heads and nk below 2^30)", what);
    UWIR_CHECK(hd > 0 && hd <= 128 && hd % 8 == 0, "%s: head size must be a multiple of 8, at most 128", what);
    UWIR_CHECK(scale >= 1e-20f && scale <= 1e20f, "%s: scale must lie in [1e-20, 1e20]", what);
    return UWIR_OK;
}

inline int xattn_check_mats(const char* what, int dtype, int hd, const XMat* in, int n_in, const XMat* out, int n_out) {
    const size_t es = dtype == UWIR_BF16 ? 2 : 4;
    auto bytes = [&](const XMat& m) { return m.rows ? ((m.rows - 1) * m.ld + (size_t)m.heads * hd) * es : 0; };
    for (int i = 0; i < n_in + n_out; ++i) {
        const XMat& m = i < n_in ? in[i] : out[i - n_in];
        if (m.rows == 0) continue;
        UWIR_CHECK(m.p, "%s: null pointer (%s)", what, m.name);
        UWIR_CHECK(m.ld >= (size_t)m.heads * hd, "%s: row stride of %s is below heads * hd", what, m.name);
        UWIR_CHECK(m.ld * es < (1u << 25), "%s: row stride of %s is 32 MB or more", what, m.name);
        UWIR_CHECK(((uintptr_t)m.p & 15) == 0 && (m.ld * es) % 16 == 0, "%s: rows of %s must be 16-byte aligned", what, m.name);
    }
    // an output may share a wider matrix with another operand (column ranges that do not meet), but no element
    for (int o = 0; o < n_out; ++o)
        for (int i = 0; i < n_in + o; ++i) {
            const XMat &a = out[o], &b = i < n_in ? in[i] : out[i - n_in];
            const size_t na = bytes(a), nb = bytes(b), wa = (size_t)a.heads * hd * es, wb = (size_t)b.heads * hd * es;
            const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
            if (!na || !nb || x + na <= y || y + nb <= x) continue;
            const size_t ld = a.ld * es;
            const size_t d = x >= y ? (x - y) % ld : (ld - (y - x) % ld) % ld;   // a's first column, seen from b's
            UWIR_CHECK(a.ld == b.ld && d >= wb && d + wa <= ld, "%s: %s overlaps %s", what, a.name, b.name);
        }
    return UWIR_OK;
}

// Memory that a call writes beside its matrices (workspace, lse) must not meet any of them.
inline int xattn_check_apart(const char* what, const char* name, const void* p, size_t n, int dtype, int hd, const XMat* m, int count) {
    const size_t es = dtype == UWIR_BF16 ? 2 : 4;
    const uintptr_t x = (uintptr_t)p;
    if (p && n)
        for (int i = 0; i < count; ++i) {
            if (!m[i].rows) continue;
            const uintptr_t y = (uintptr_t)m[i].p;
            const size_t nb = ((m[i].rows - 1) * m[i].ld + (size_t)m[i].heads * hd) * es;
            UWIR_CHECK(x + n <= y || y + nb <= x, "%s: %s overlaps %s", what, name, m[i].name);
        }
    return UWIR_OK;
}

// key_lens and key_mask are read while the call writes: neither may meet an output, nor the memory `extra` written beside them.
struct XRange {
    const void* p;
    size_t n;
    const char* name;
};
inline int xattn_check_keys(const char* what, const int* lens, const unsigned char* mask, size_t ldm, int B, int nk, int dtype, int hd,
                            const XMat* out, int n_out, const XRange* extra, int n_extra) {
    const XRange in[] = {{lens, (size_t)B * sizeof(int), "key_lens"}, {mask, nk ? (size_t)(B - 1) * ldm + nk : 0, "key_mask"}};
    for (const XRange& r : in) {
        if (!r.p || !r.n) continue;
        if (int rc = xattn_check_apart(what, r.name, r.p, r.n, dtype, hd, out, n_out)) return rc;
        for (int i = 0; i < n_extra; ++i) {
            const uintptr_t x = (uintptr_t)r.p, y = (uintptr_t)extra[i].p;
            UWIR_CHECK(!extra[i].p || !extra[i].n || x + r.n <= y || y + extra[i].n <= x, "%s: %s overlaps %s", what, extra[i].name, r.name);
        }
    }
    return UWIR_OK;
}

}  // namespace
