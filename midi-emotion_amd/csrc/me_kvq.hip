// Quantised key / value cache (gfx950): rows written as 4-bit e2m1 or 8-bit e4m3 codes with one bfloat16 scale, read back, and the
// attention of one new query per (sequence, head) against them.
//
// 4 bits: the codes are what the matrix instructions of this part multiply directly (v_mfma_f32_16x16x128_f8f6f4 takes e2m1
// operands), so neither K nor V is ever unpacked: a lane's 16 bytes from memory (32 codes) ARE its operand.  What has to be converted
// is the other side, the query once per call and the softmax weights once per key: scaled by a power of two, they are written in
// base 32, x = d0 + d1 / 32 + d2 / 1024 + ..., with whole digits -16 .. 16 that e4m3 holds exactly, and the digits take the rows of the 16-row
// operand that a single query leaves idle.  Whole digits, because that unit does not add in 32 bits: with e4m3 numbers
// of all sizes it lost up to 2^-11 of the largest product (measured).  Digit times code is a multiple of 1/2 below 97, so
// its sums are exact.  Four digits leave 2^-19 of the largest value, six (f32) 2^-29.
// 8 bits: e4m3 codes span 2^17, so they are widened to bfloat16 (exactly, two per instruction) for the bf16 product, which adds in
// 32 bits; the query (scaled by a power of two too) and the weights enter as one to three bfloat16 parts, again in the idle rows.
//
// Layout of a block of 32 tokens (one head), in the order of the operands; a code's position counts codes:
//   K: the contraction runs over dh, so 32 of a row's codes form a lane's chunk.  4 bits: chunk (group, lane) at (group * 16 + lane) * 32
//      dh 64: group = 2 (token / 16) + d / 32;  dh 32: group = token / 16;  lane = token % 16
//      dh 48: dimensions 0..31 in group 2 (token / 16), dimensions 32..47 in group 1, second half of the chunk for tokens 16..31
//   V: the contraction runs over tokens: 4 bits: code (token, d) at d * 32 + token
//   8 bits: the same chunks of 32 codes, but a lane takes them as two pieces of 16: all first pieces, then all second ones.
#include "me_common.h"
#include <algorithm>
#include <math.h>

namespace {

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef unsigned short u16;

constexpr int KB = 32;                                        // tokens per block

template <int BITS, int DH> struct Fmt {
    static constexpr int BLK = KB * DH * BITS / 8;            // bytes of a block (K and V alike)
    static constexpr float TOP = BITS == 4 ? 6.f : 448.f;     // largest value of the code's type
};

// byte offset, inside a K block, of the codes of dimensions d .. d + 7 (d % 8 == 0) of token tk: 4 (8) consecutive bytes
template <int BITS, int DH> ME_DEV int k_byte(int tk, int d) {
    const int lane = tk & 15, half = tk >> 4;
    int group, i;
    if (DH == 64) { group = 2 * half + (d >> 5); i = d & 31; }
    else if (DH == 32) { group = half; i = d; }
    else if (d < 32) { group = 2 * half; i = d; }
    else { group = 1; i = 16 * half + d - 32; }
    if (BITS == 4) return (group * 16 + lane) * 16 + (i >> 1);
    return (i >> 4) * (DH / 16 * 256) + (group * 16 + lane) * 16 + (i & 15);
}
// byte offset, inside a V block, of the codes of tokens tk .. tk + 7 (tk % 8 == 0) of dimension d
template <int BITS, int DH> ME_DEV int v_byte(int tk, int d) {
    if (BITS == 4) return d * 16 + (tk >> 1);
    return (tk >> 4) * (DH * 16) + d * 16 + (tk & 15);
}

// first position of the call (all sequences alike, or one value for each)
ME_DEV int pos_of(int t, const int32_t* t_dev, int ld_t, int b) { return t_dev ? t_dev[(size_t)b * ld_t] : t; }

struct RowArgs {                                              // k / v rows [B][n][H][dh], strides in elements, dh contiguous
    void* k; void* v;
    int64_t skb, skn, skh, svb, svn, svh;
    uint8_t* kc; u16* ks; uint8_t* vc; u16* vs;
    int n, H, blocks, t, ld_t;
    const int32_t* t_dev; const int32_t* lens;
};

// 8 elements of a row: VEC = two (four) 16-byte accesses, for rows that are 16-byte aligned throughout
template <typename T, bool VEC> ME_DEV void load8(float (&x)[8], const T* p) {
    constexpr int CH = ET<T>::CH;
    if constexpr (VEC) {
#pragma unroll
        for (int u = 0; u < 8 / CH; ++u) {
            const chunk16 c = ld_chunk(p + u * CH);
            const T* e = reinterpret_cast<const T*>(&c);
#pragma unroll
            for (int i = 0; i < CH; ++i) x[u * CH + i] = ET<T>::to_f(e[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = ET<T>::to_f(p[i]);
    }
}
template <typename T, bool VEC> ME_DEV void store8(T* p, const float (&x)[8]) {
    if constexpr (!VEC) {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = ET<T>::from_f(x[i]);
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<f32x4_t*>(p) = (f32x4_t){x[0], x[1], x[2], x[3]};
        *reinterpret_cast<f32x4_t*>(p + 4) = (f32x4_t){x[4], x[5], x[6], x[7]};
    } else {
        typename V16<T>::x8 v;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (T)x[i];
        *reinterpret_cast<typename V16<T>::x8*>(p) = v;
    }
}

// One row spread over 8 lanes (8 values each): the row's scale and the lane's 8 codes (32 or 64 bits).
// scale = cut_to_bfloat16(amax / TOP): cut, not rounded, so that TOP * scale (amax and a bit at most) never leaves T's range; what lies above
// TOP * scale (by at most 2^-7 of it) takes the largest code.  The codes are those of the held scale, so cutting it costs no accuracy
// beyond that.  The quotient is correctly rounded (one Newton step from the rounded reciprocal): where x / scale is exactly half
// way between two codes it comes out exactly, and the conversion's ties-to-even decides.  f32 rows have quotients nearer to such a border than
// a rounding step; there an inexact quotient with an even last bit is moved by one bit toward the true one, off the border.
template <int BITS, bool WIDE> ME_DEV void quantise8(const float (&x)[8], u16& scale, uint32_t (&codes)[2], bool active) {
    constexpr float TOP = BITS == 4 ? 6.f : 448.f;
    uint32_t am = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) am = max(am, __float_as_uint(x[i]) & 0x7fffffffu);     // a NaN is larger than any number here
    if (!active) am = 0;
    am = max(am, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)am, 0xB1, 0xF, 0xF, true));
    am = max(am, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)am, 0x4E, 0xF, 0xF, true));
    am = max(am, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)am, 0x141, 0xF, 0xF, true));
    const float amax = __uint_as_float(am);
    const bool fine = am < 0x7f800000u, kept = fine && amax >= 0x1p-96f;
    // amax / TOP as torch divides by a number on this device: times its rounded reciprocal.  After the cut that is the quotient's for every bf16
    // and f16 amax; of the f32 ones, 42 (TOP 6) or 55 (TOP 448) mantissas of 2^23, one bit below TOP * scale, get that scale instead of the next lower
    constexpr float RT = 1.f / TOP;
    const uint32_t sb = __float_as_uint(amax * RT) & 0xffff0000u;
    scale = fine ? (kept ? (u16)(sb >> 16) : (u16)0) : (u16)0x7fc0;
    // 1 / s, correctly rounded for the 8 significant bits of a scale (all of them checked): hardware estimate and one Newton step
    const float s = kept ? __uint_as_float(sb) : 1.f, r0 = __builtin_amdgcn_rcpf(s), r = fmaf(fmaf(-s, r0, 1.f), r0, r0);
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float q0 = x[i] * r;
        float q = fmaf(fmaf(-q0, s, x[i]), r, q0);
        if (WIDE) {
            const float rem = fmaf(-q, s, x[i]);
            const uint32_t qb = __float_as_uint(q);
            if (rem != 0.f && !(qb & 1u)) q = __uint_as_float(((__float_as_uint(rem) ^ qb) >> 31) ? qb - 1u : qb + 1u);
        }
        y[i] = fminf(fmaxf(q, -TOP), TOP);
    }
    if (BITS == 4) {
        uint32_t c = 0;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[0], y[1], 1.f, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[2], y[3], 1.f, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[4], y[5], 1.f, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[6], y[7], 1.f, 3);
        codes[0] = kept ? c : 0;
        codes[1] = 0;
    } else {
        int c0 = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false), c1 = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
        codes[0] = kept ? (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], c0, true) : 0;
        codes[1] = kept ? (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], c1, true) : 0;
    }
}

// ---------------------------------------------------------------------------------------------------------
// write: block = one 32-token block of one (sequence, head): 8 lanes per row, so that a row's maximum takes three lane
// exchanges and its 16-bit values one 16-byte load per lane.  Bounded by memory where there is enough of it: 32 x 2048 x 8 rows of 64 in
// bf16, 4 bits: 33.8 us = 5.0 TB/s of K, V, codes and scales moved (a copy reaches 5.0); 64 x 8 rows (a step): 3.7 us, a launch's latency.  K goes straight to its chunk (4 / 8 bytes per
// lane); V changes its order through LDS (8 tokens of a dimension per thread), and a group of 8 tokens that the call covers only in
// part keeps its other codes (read, merged, written by the one thread that owns the word).
// ---------------------------------------------------------------------------------------------------------
template <typename T, int BITS, int DH, bool VEC>
__global__ __launch_bounds__(256) void kvq_write_kernel(const RowArgs a) {
    constexpr int W = BITS == 4 ? 1 : 2;
    __shared__ uint32_t vq[KB][8 * W];
    const int tid = threadIdx.x, key = tid >> 3, sub = tid & 7, h = blockIdx.y, b = blockIdx.z;
    const int t = pos_of(a.t, a.t_dev, a.ld_t, b);
    if (t < 0 || t >= a.blocks * KB) return;                  // block-uniform: a sequence that does not begin in the cache is left out
    const int nb = a.lens ? min(a.n, a.lens[b]) : a.n;
    const int end = (int)min((int64_t)t + nb, (int64_t)a.blocks * KB);
    const int blk = t / KB + blockIdx.x, j0 = blk * KB;
    if (j0 >= end) return;
    const int j = j0 + key, d0 = sub * 8;
    const bool valid = j >= t && j < end, active = valid && d0 < DH;
    float xk[8], xv[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) { xk[i] = 0.f; xv[i] = 0.f; }
    if (active) {
        const int64_t i = j - t;
        load8<T, VEC>(xk, reinterpret_cast<const T*>(a.k) + (int64_t)b * a.skb + i * a.skn + (int64_t)h * a.skh + d0);
        load8<T, VEC>(xv, reinterpret_cast<const T*>(a.v) + (int64_t)b * a.svb + i * a.svn + (int64_t)h * a.svh + d0);
    }
    u16 sk, sv;
    uint32_t ck[2], cv[2];
    quantise8<BITS, sizeof(T) == 4>(xk, sk, ck, active);
    quantise8<BITS, sizeof(T) == 4>(xv, sv, cv, active);
    const size_t bh = (size_t)b * a.H + h;
    uint8_t* kb = a.kc + (bh * a.blocks + blk) * Fmt<BITS, DH>::BLK;
    uint8_t* vb = a.vc + (bh * a.blocks + blk) * Fmt<BITS, DH>::BLK;
    if (active) {
        uint32_t* p = reinterpret_cast<uint32_t*>(kb + k_byte<BITS, DH>(key, d0));
        p[0] = ck[0];
        if (W == 2) p[1] = ck[1];
    }
    if (valid && sub == 0) { a.ks[bh * a.blocks * KB + j] = sk; a.vs[bh * a.blocks * KB + j] = sv; }
#pragma unroll
    for (int w = 0; w < W; ++w) vq[key][sub * W + w] = cv[w];
    __syncthreads();
    const int d = tid >> 2, q = tid & 3;                      // 8 tokens 8 q .. 8 q + 7 of dimension d
    if (d >= DH) return;
    uint32_t* p = reinterpret_cast<uint32_t*>(vb + v_byte<BITS, DH>(8 * q, d));
    const int at = BITS == 4 ? 4 * (d & 7) : 8 * (d & 3), col = BITS == 4 ? d >> 3 : d >> 2;
    uint32_t word[W], c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = __builtin_amdgcn_ubfe(vq[8 * q + i][col], at, BITS);
#pragma unroll
    for (int w = 0; w < W; ++w) {
        word[w] = c[(8 / W) * w];
#pragma unroll
        for (int i = 1; i < 8 / W; ++i) word[w] |= c[(8 / W) * w + i] << (BITS * i);
    }
    if (t <= j0 && end >= j0 + KB) {                          // block-uniform: the call covers the block
#pragma unroll
        for (int w = 0; w < W; ++w) p[w] = word[w];
        return;
    }
    const int lo = max(0, t - (j0 + 8 * q)), hi = min(8, end - (j0 + 8 * q));
    if (lo >= hi) return;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const int a0 = max(lo - (8 / W) * w, 0), a1 = min(hi - (8 / W) * w, 8 / W);
        if (a0 >= a1) continue;
        const uint32_t mask = (a1 * BITS == 32 ? 0xffffffffu : (1u << (a1 * BITS)) - 1u) & ~((1u << (a0 * BITS)) - 1u);
        p[w] = mask == 0xffffffffu ? word[w] : (p[w] & ~mask) | (word[w] & mask);
    }
}

// ---------------------------------------------------------------------------------------------------------
// read back: the same split (27.3 us = 6.2 TB/s for the rows above: mostly stores); a row behind the sequence's length (or the cache's end) reads as zeros
// ---------------------------------------------------------------------------------------------------------
template <int BITS> ME_DEV void expand8(float (&x)[8], uint32_t c0, uint32_t c1, float s) {
    f32x2_t r[4];
    if (BITS == 4) {
        r[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c0, 1.f, 0);
        r[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c0, 1.f, 1);
        r[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c0, 1.f, 2);
        r[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c0, 1.f, 3);
    } else {
        r[0] = __builtin_amdgcn_cvt_pk_f32_fp8((int)c0, false);
        r[1] = __builtin_amdgcn_cvt_pk_f32_fp8((int)c0, true);
        r[2] = __builtin_amdgcn_cvt_pk_f32_fp8((int)c1, false);
        r[3] = __builtin_amdgcn_cvt_pk_f32_fp8((int)c1, true);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = r[i >> 1][i & 1] * s;
}
ME_DEV float bf16_bits(u16 u) { return __uint_as_float((uint32_t)u << 16); }

template <typename T, int BITS, int DH, bool VEC>
__global__ __launch_bounds__(256) void kvq_read_kernel(const RowArgs a) {
    constexpr int W = BITS == 4 ? 1 : 2;
    __shared__ uint32_t vq[8][8][4 * W];                      // [d % 8][d / 8][tokens]: the 8 lanes of a row read 8 different banks
    const int tid = threadIdx.x, key = tid >> 3, sub = tid & 7, h = blockIdx.y, b = blockIdx.z;
    const int t = pos_of(a.t, a.t_dev, a.ld_t, b);
    const int nb = a.lens ? max(0, min(a.n, a.lens[b])) : a.n;
    // blocks of the cache counted from the one that holds t; a sequence whose t lies outside reads as zeros from its row 0 on
    const bool in = t >= 0 && t < a.blocks * KB;
    const int first = in ? t : 0;
    const int blk = first / KB + blockIdx.x, j = blk * KB + key;
    const int64_t i = (int64_t)j - first;
    const bool held = in && i >= 0 && i < nb && j < a.blocks * KB;
    const size_t bh = (size_t)b * a.H + h;
    const int d0 = sub * 8;
    float xk[8], xv[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) { xk[e] = 0.f; xv[e] = 0.f; }
    if (in && blk < a.blocks) {                               // block-uniform
        const uint8_t* kb = a.kc + (bh * a.blocks + blk) * Fmt<BITS, DH>::BLK;
        const uint8_t* vb = a.vc + (bh * a.blocks + blk) * Fmt<BITS, DH>::BLK;
        const int d = tid >> 2, q = tid & 3;
        if (d < DH) {
            const uint32_t* p = reinterpret_cast<const uint32_t*>(vb + v_byte<BITS, DH>(8 * q, d));
#pragma unroll
            for (int w = 0; w < W; ++w) vq[d & 7][d >> 3][q * W + w] = p[w];
        }
        uint32_t c0 = 0, c1 = 0;
        float sk = 0.f, sv = 0.f;
        if (held && d0 < DH) {
            const uint32_t* p = reinterpret_cast<const uint32_t*>(kb + k_byte<BITS, DH>(key, d0));
            c0 = p[0];
            if (W == 2) c1 = p[1];
            sk = bf16_bits(a.ks[bh * a.blocks * KB + j]);
            sv = bf16_bits(a.vs[bh * a.blocks * KB + j]);
        }
        __syncthreads();
        if (held && d0 < DH) {
            expand8<BITS>(xk, c0, c1, sk);
            uint32_t v0 = 0, v1 = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t w = vq[e][sub][(key >> 3) * W + (W == 2 ? (key >> 2) & 1 : 0)];
                if (BITS == 4) v0 |= ((w >> (4 * (key & 7))) & 15u) << (4 * e);
                else { const uint32_t c = (w >> (8 * (key & 3))) & 255u; if (e < 4) v0 |= c << (8 * e); else v1 |= c << (8 * (e - 4)); }
            }
            expand8<BITS>(xv, v0, v1, sv);
        }
    }
    if (i < 0 || i >= a.n || d0 >= DH) return;
    store8<T, VEC>(reinterpret_cast<T*>(a.k) + (int64_t)b * a.skb + i * a.skn + (int64_t)h * a.skh + d0, xk);
    store8<T, VEC>(reinterpret_cast<T*>(a.v) + (int64_t)b * a.svb + i * a.svn + (int64_t)h * a.svh + d0, xv);
}

// ---------------------------------------------------------------------------------------------------------
// attention: a block is up to 8 waves = heads x key ranges of one sequence; keys in tiles of 128, a head's ranges take them in turn and
// meet in LDS at the end; grid.x may cut the keys further
//   s_j = (q.k_j + q.E[M-1-(t-j)]) / sqrt(dh);  running maximum and sum in base 2, 32 bits
//   K: two MFMAs give a lane the four row products of ONE key (rows 4 g + i of the result: digit i, and A's zero blocks pick
//      the chunk that belongs to the row's 16 keys); V: the weights p_j * scale_j (4 bits: scaled by a power of two per tile) are the rows.
//   E is shared by a block's heads: its products for a stretch of keys come from one matrix product per 16 keys and wait in LDS.
// What bounds it: long caches the memory, 64 x 8 heads x 16384 keys of 64 in 4 bits 97 us = 5.9 TB/s; with the relative products and a
// mask, 64 x 16 x 1999 of 48 in 8 bits (ragged), 42 us = 4.3 TB/s; with them alone, 64 x 8 x 2048 of 64 in 4 bits, 23 us = 3.1 TB/s: a block's
// products precede its stream.  Few rows: the chain of latencies, 1 x 8 x 256: 5.7 us, 4 x 8 x 2048: 8.3 us with its join, where 4.5 MB would
// take 0.9.  With the step's rows written too 0.9 .. 1.6 us more (64 x 16 x 1999: 2.9); without the join, as a decode step calls it, 6.1 and 7.6.
// A tile of 128 keys is two K operands' columns of 64 lanes (a lane holds two logits) and one V operand's depth, and the next tile's loads are in flight under a tile's products.
// ---------------------------------------------------------------------------------------------------------
constexpr int RELS = 4096;                                    // relative logits in LDS: a stretch of RELS / (heads of the block) keys
constexpr int TK = 128;                                       // keys per tile
template <int BITS> constexpr int PROW = BITS == 4 ? TK + 16 : 2 * TK + 16;   // bytes between the parts in LDS (16 more than the row: other banks)
constexpr int WAVES = 8;                                      // waves of a block at most: heads x key ranges, both powers of two
constexpr int HG = 8;                                         // heads of a block at most

struct AttnArgs {
    const void* q; int64_t sqb, sqh;
    const uint8_t* kc; const u16* ks; const uint8_t* vc; const u16* vs;
    const void* E; int M;
    const uint8_t* pad; int ld_pad;
    void* out; int64_t sob, soh;
    float* part; int nsplit;
    const void* kn; const void* vn; int64_t snb, snh;         // the rows of position t itself, still to be cached (or NULL)
    int H, blocks, t, ld_t, hpb, kw;
    const int32_t* t_dev;
    float scale;
    float munit;                                              // unit of a record's maximum: 1 = base 2 (kvq_join_kernel), ln 2 = natural
};

template <int BITS, int DH> struct Tile {
    static constexpr int NK = DH == 32 ? 2 : 4;               // K operands (64 keys each at dh 32, 32 keys otherwise)
    static constexpr int NV = DH / 16;                        // V operands (16 dimensions each)
    static constexpr int P = BITS == 4 ? 1 : 2;               // 16-byte pieces per operand and lane
    u32x4_t k[NK][P], v[NV][P];
    u16 ks[2], vs[2];
    uint8_t pad[2];
};

template <int BITS, int DH>
ME_DEV void load_tile(Tile<BITS, DH>& x, const uint8_t* kc, const uint8_t* vc, const u16* ks, const u16* vs, const uint8_t* pad, int ld_pad, int jt, int j1, int lane) {
    typedef Tile<BITS, DH> TL;
    constexpr int BLK = Fmt<BITS, DH>::BLK, GB = DH / 16 * 256;             // GB: bytes of all first pieces of a K block
    const u32x4_t zero = {0u, 0u, 0u, 0u};
    const int kb = jt / KB, c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int u = 0; u < TL::NK; ++u) {
        const int blk = DH == 32 ? kb + 2 * u + (lane >> 5) : kb + u;
        const int at = DH == 32 ? (lane & 31) * 16 : lane * 16;
        const bool ok = blk * KB < j1 && (DH != 48 || lane < 48);
        const uint8_t* p = kc + (size_t)blk * BLK + at;
#pragma unroll
        for (int s = 0; s < TL::P; ++s) x.k[u][s] = ok ? *reinterpret_cast<const u32x4_t*>(p + s * GB) : zero;
    }
    const bool okv = (kb + g) * KB < j1;
    const uint8_t* pv = vc + (size_t)(kb + g) * BLK + c * 16;
#pragma unroll
    for (int u = 0; u < TL::NV; ++u)
#pragma unroll
        for (int s = 0; s < TL::P; ++s) x.v[u][s] = okv ? *reinterpret_cast<const u32x4_t*>(pv + u * 256 + s * (DH * 16)) : zero;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int j = jt + 64 * u + lane;
        const bool ok = j < j1;
        x.ks[u] = ok ? ks[j] : (u16)0;
        x.vs[u] = ok ? vs[j] : (u16)0;
        x.pad[u] = ok ? (pad && j < ld_pad ? pad[j] : (uint8_t)0) : (uint8_t)1;
    }
}

// A = digits (32 bytes per lane), B = 4-bit codes; all block scales 1: the form without scale operands
ME_DEV f32x4_t mma_codes(const i32x8_t& a, const u32x4_t& b, const f32x4_t& c) {
    const i32x8_t w = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, w, c, 0, 4, 0, 0, 0, 0);
}
// 8 e4m3 codes as bfloat16
ME_DEV bf16x8_t widen8(uint32_t c0, uint32_t c1) {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c0, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c0, 1.f, true);
    const auto c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c1, 1.f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c1, 1.f, true);
    return (bf16x8_t){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// e4m3 codes that are no numbers (0x7f, 0xff; never written, but memory that was never written may hold them) become zeros
ME_DEV void numbers(u32x4_t& x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t m = ((x[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
        x[i] &= ~(m - (m >> 7));
    }
}
ME_DEV f32x4_t mma_bf16(const bf16x8_t& a, const bf16x8_t& b, const f32x4_t& c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
ME_DEV void lds_order() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }      // a wave's own LDS writes, then its reads
ME_DEV i32x8_t two_pieces(const u32x4_t& lo, const u32x4_t& hi) {
    return (i32x8_t){(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}
// power of two f with x f in [8, 16) (x > 0), and 1 / f
ME_DEV void unit(float x, float& f, float& inv) {
    const int e = min(254, max(8, (int)(__float_as_uint(x) >> 23)));
    f = __uint_as_float((uint32_t)(257 - e) << 23);
    inv = __uint_as_float((uint32_t)(e - 3) << 23);
}
// sums of the rows' products: digits d0 + d1 / 32 + d2 / 32^2 + d3 / 32^3, parts d0 + d1 + d2
ME_DEV float join_digits(const f32x4_t& d) { return fmaf(fmaf(fmaf(d[3], 0x1p-5f, d[2]), 0x1p-5f, d[1]), 0x1p-5f, d[0]); }

// operand row of the query: the B operand's slot (group sg, code i) holds which dimension for the 16 keys of row r; -1 = none of theirs
template <int DH> ME_DEV int slot_dim(int r, int sg, int i) {
    if (DH == 32) return sg == (r >> 2) ? i : -1;
    const int half = (r >> 2) & 1;
    if (DH == 64) return (sg >> 1) == half ? (sg & 1) * 32 + i : -1;
    if (sg == 2 * half) return i;
    return sg == 1 && (i >> 4) == half ? 32 + (i & 15) : -1;
}

// a row's operand (one of 16 rows, lane group g's share of the contraction) of the relative product q E^T in T
template <typename T, int DH> struct EFrag {
    static constexpr int N = (DH + 31) / 32;
    typename V16<T>::x8 v[N];
    ME_DEV void load(const T* p, int g) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            v[k] = (typename V16<T>::x8){0, 0, 0, 0, 0, 0, 0, 0};
            if (32 * k + 8 * g < DH) v[k] = *reinterpret_cast<const typename V16<T>::x8*>(p + 32 * k + 8 * g);
        }
    }
    ME_DEV void set(const float* p, int g) {
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[k][i] = 32 * k + 8 * g < DH ? (T)p[32 * k + 8 * g + i] : (T)0.f;
    }
    ME_DEV static f32x4_t mma(const EFrag& x, const EFrag& y) {
        f32x4_t d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if constexpr (__is_same(T, bf16_t)) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.v[k], y.v[k], d, 0, 0, 0);
            else d = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.v[k], y.v[k], d, 0, 0, 0);
        }
        return d;
    }
};
template <int DH> struct EFrag<float, DH> {                   // group g takes a quarter of the row
    f32x4_t v[DH / 16];
    ME_DEV void load(const float* p, int g) {
#pragma unroll
        for (int k = 0; k < DH / 16; ++k) v[k] = *reinterpret_cast<const f32x4_t*>(p + g * (DH / 4) + 4 * k);
    }
    ME_DEV void set(const float* p, int g) { load(p, g); }
    ME_DEV static f32x4_t mma(const EFrag& x, const EFrag& y) {
        f32x4_t d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < DH / 4; ++k) d = __builtin_amdgcn_mfma_f32_16x16x4f32(x.v[k >> 2][k & 3], y.v[k >> 2][k & 3], d, 0, 0, 0);
        return d;
    }
};

template <typename T, int BITS, int DH, bool REL>
__global__ __launch_bounds__(64 * WAVES) void kvq_attn_kernel(const AttnArgs a) {
    constexpr bool WIDE = sizeof(T) == 4;
    constexpr int NP = BITS == 4 ? (WIDE ? 6 : 4) : (WIDE ? 3 : 2);               // digits / bfloat16 parts of a weight
    constexpr int NQ = BITS == 4 ? NP : (WIDE ? 3 : (__is_same(T, bf16_t) ? 1 : 2));      // and of a query element (16-bit types: exact in parts)
    constexpr int NS = BITS == 4 && WIDE ? 2 : 1;             // operand sets of four rows
    constexpr int PR = PROW<BITS>;
    constexpr float LOG2E = 1.4426950408889634f;
    __shared__ __attribute__((aligned(16))) float qs[HG][DH];
    __shared__ __attribute__((aligned(16))) uint8_t parts[WAVES][NP * PR];
    __shared__ float rel[REL ? RELS : 1];
    __shared__ float jm[WAVES], jl[WAVES], jo[WAVES][DH];     // key ranges of a head meet here
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), nw = blockDim.x >> 6;
    const int c = lane & 15, g = lane >> 4;
    const int hpb = a.hpb, kw = a.kw, hw = wid / kw, wk = wid % kw;
    const int split = blockIdx.x, b = blockIdx.z, h0 = blockIdx.y * hpb, nh = min(hpb, a.H - h0);
    const int hh = min(hw, nh - 1), h = h0 + hh;              // waves past the last head repeat it and store nothing
    const int t = pos_of(a.t, a.t_dev, a.ld_t, b);
    const bool fresh = a.kn && t >= 0 && t < a.blocks * KB;   // position t comes with the call; the keys before it are in the cache
    const int n = fresh ? t : max(min(t, a.blocks * KB - 1) + 1, 0);
    const int last = fresh ? t : n - 1;                       // the query's position
    const int per = ((n + a.nsplit - 1) / a.nsplit + TK - 1) / TK * TK;
    const int j0 = (int)min((int64_t)split * per, (int64_t)n), j1 = (int)min((int64_t)j0 + per, (int64_t)n);
    const size_t bh = (size_t)b * a.H + h;
    const uint8_t* kc = a.kc + bh * a.blocks * Fmt<BITS, DH>::BLK;
    const uint8_t* vc = a.vc + bh * a.blocks * Fmt<BITS, DH>::BLK;
    const u16* ks = a.ks + bh * a.blocks * KB;
    const u16* vs = a.vs + bh * a.blocks * KB;
    const uint8_t* pad = a.pad ? a.pad + (size_t)b * a.ld_pad : nullptr;

    Tile<BITS, DH> cur;
    if (j0 + wk * TK < j1) load_tile<BITS, DH>(cur, kc, vc, ks, vs, pad, a.ld_pad, j0 + wk * TK, j1, lane);       // in flight under the query's preparation

    for (int i = tid; i < nh * DH; i += nw * 64)
        qs[i / DH][i % DH] = ET<T>::to_f(reinterpret_cast<const T*>(a.q)[(int64_t)b * a.sqb + (int64_t)(h0 + i / DH) * a.sqh + i % DH]);
    __syncthreads();

    // ---- the query as operand rows: row r carries digit / part r % 4 for the keys of row group r / 4.  dh 32: qa covers 64 keys; else
    //      qa (rows 0..7) keys 0..31 and qb (rows 8..15) keys 32..63 of a group
    uint8_t* pw = parts[wid];
    float qinv = 1.f;
    i32x8_t qa[NS], qb[NS];                                   // 4 bits
    bf16x8_t ha[4], hb[4];                                    // 8 bits: steps of 8 codes
    {
        float x = lane < DH ? qs[hh][lane] : 0.f;
        if (__builtin_amdgcn_ballot_w64(!(fabsf(x) <= 3.402823466e38f))) { qinv = __builtin_nanf(""); x = 0.f; }   // an infinity or a NaN in the query: every logit is NaN
        float f, fi;                                          // 8 bits: products with codes up to 448 stay inside f32 whatever the query's size
        unit(wave_max(fabsf(x)), f, fi);
        qinv *= fi;
        x *= f;
        if constexpr (BITS == 4) {
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
                const float d = rintf(x);
                if (lane < DH) pw[i * PR + lane] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(d, d, 0, false);
                x = (x - d) * 32.f;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
                const bf16_t d = (bf16_t)x;
                if (lane < DH) reinterpret_cast<bf16_t*>(pw + i * PR)[lane] = d;
                x -= (float)d;
            }
        }
    }
    lds_order();
    const u32x4_t zero = {0u, 0u, 0u, 0u};
    if constexpr (BITS == 4) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int digit = 4 * s + (c & 3);
            u32x4_t pc[2];
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                // the e4m3 operand's pieces are k = 16 g .. and 64 + 16 g .., the e2m1 operand's lane has k = 32 g .. (measured on this part)
                const int dm = slot_dim<DH>(c, 2 * p + (g >> 1), 16 * (g & 1));
                pc[p] = dm >= 0 && digit < NQ ? *reinterpret_cast<const u32x4_t*>(pw + digit * PR + dm) : zero;
            }
            const i32x8_t w = two_pieces(pc[0], pc[1]), z = two_pieces(zero, zero);
            qa[s] = DH == 32 || c < 8 ? w : z;
            qb[s] = c < 8 ? z : w;
        }
    } else {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int dm = slot_dim<DH>(c, g, 8 * s);
            const u32x4_t w = dm >= 0 && (c & 3) < NQ ? *reinterpret_cast<const u32x4_t*>(pw + (c & 3) * PR + 2 * dm) : zero;
            ha[s] = __builtin_bit_cast(bf16x8_t, DH == 32 || c < 8 ? w : zero);
            hb[s] = __builtin_bit_cast(bf16x8_t, c < 8 ? zero : w);
        }
    }
    lds_order();

    float m = -INFINITY, lsum = 0.f, acc[DH / 16];
#pragma unroll
    for (int u = 0; u < DH / 16; ++u) acc[u] = 0.f;
    const float cs = a.scale * LOG2E, cq = cs * qinv;

    // ---- position t itself: quantised into the cache by the first range's wave (lanes 0..7 K, 8..15 V: 8 values each), which starts its
    //      softmax with it, from the held values in 32 bits -- the cache is not read where this launch writes it
    if (fresh && split == 0 && wk == 0 && hw < nh) {
        const int sub = lane & 7, d0 = sub * 8, tk = t & (KB - 1);
        const bool isv = lane >= 8, on = lane < 16 && d0 < DH;
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = 0.f;
        if (on) load8<T, true>(x, reinterpret_cast<const T*>(isv ? a.vn : a.kn) + (int64_t)b * a.snb + (int64_t)h * a.snh + d0);
        u16 sc;
        uint32_t cd[2];
        quantise8<BITS, WIDE>(x, sc, cd, on);
        const size_t blk = (size_t)(t / KB) * Fmt<BITS, DH>::BLK;
        if (on && !isv) {
            uint32_t* p = reinterpret_cast<uint32_t*>(const_cast<uint8_t*>(kc) + blk + k_byte<BITS, DH>(tk, d0));
            p[0] = cd[0];
            if (BITS == 8) p[1] = cd[1];
        }
        if (on && isv) {
            uint8_t* p = const_cast<uint8_t*>(vc) + blk + (BITS == 4 ? tk >> 1 : (tk >> 4) * (DH * 16) + (tk & 15)) + d0 * 16;
            if (BITS == 4) {
                uint32_t old[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) old[i] = p[16 * i];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t cc = (cd[0] >> (4 * i)) & 15u;
                    p[16 * i] = (uint8_t)(tk & 1 ? (old[i] & 15u) | (cc << 4) : (old[i] & 0xf0u) | cc);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) p[16 * i] = (uint8_t)(cd[i >> 2] >> (8 * (i & 3)));
            }
        }
        if (lane == 0) const_cast<u16*>(ks)[t] = sc;
        if (lane == 8) const_cast<u16*>(vs)[t] = sc;
        expand8<BITS>(x, cd[0], cd[1], bf16_bits(sc));
        float s = 0.f;
        if (on && !isv) {
            float e[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if constexpr (REL) load8<T, true>(e, reinterpret_cast<const T*>(a.E) + (size_t)(a.M - 1) * DH + d0);
#pragma unroll
            for (int i = 0; i < 8; ++i) s = fmaf(qs[hh][d0 + i], x[i] + e[i], s);
        }
        if (on && isv) {
#pragma unroll
            for (int i = 0; i < 8; ++i) jo[wid][d0 + i] = x[i];
        }
        s = wave_sum(s) * cs + (qinv - qinv);                 // NaN with a query that is none
        lds_order();
        if (!(pad && t < a.ld_pad && pad[t]) && s != -INFINITY) {
            const float one = __builtin_amdgcn_exp2f(s - s);  // 1, or NaN where the logit is none
            m = s;
            lsum = lane == 0 ? one : 0.f;
#pragma unroll
            for (int u = 0; u < DH / 16; ++u) acc[u] = one * jo[wid][16 * u + (lane & 15)];
        }
        lds_order();
    }

    EFrag<T, DH> eq;                                          // row c: the query of the block's head c (rows past the last repeat it)
    if constexpr (REL) eq.set(qs[min(c, nh - 1)], g);
    const int stretch = REL ? RELS / hpb : max(j1 - j0, 1);   // a multiple of kw tiles
    for (int c0 = j0; c0 < j1; c0 += stretch) {
        const int c1 = min(c0 + stretch, j1);
        if constexpr (REL) {
            __syncthreads();                                  // the last stretch has been read
            constexpr int U = BITS == 4 ? 4 : 2;              // key groups of 16 in flight per wave (8 bits: four would spill)
            for (int k0 = wid * 16; k0 < c1 - c0; k0 += nw * 16 * U) {
                EFrag<T, DH> e[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int row = a.M - 1 - last + min(c0 + k0 + u * nw * 16 + c, last);
                    e[u].load(reinterpret_cast<const T*>(a.E) + (size_t)row * DH, g);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int kt = k0 + u * nw * 16;
                    const f32x4_t d = EFrag<T, DH>::mma(eq, e[u]);
                    if (kt < c1 - c0) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) if (4 * g + i < nh) rel[(4 * g + i) * stretch + kt + c] = d[i];
                    }
                }
            }
            __syncthreads();
        }
        for (int jt = c0 + wk * TK; jt < c1; jt += kw * TK) {
            Tile<BITS, DH> nxt;
            const bool more = jt + kw * TK < j1;
            if (more) load_tile<BITS, DH>(nxt, kc, vc, ks, vs, pad, a.ld_pad, jt + kw * TK, j1, lane);
            // 8 bits: a code meets the other rows' zeros in the products, so a code that is no number, in a row that is left out, would reach
            // other rows.  Seen in the result (two comparisons a tile, where cleaning all codes first cost 8 %), and done again without
            const bool holes = BITS == 8 && __builtin_amdgcn_ballot_w64(cur.pad[0] | cur.pad[1]);
            // ---- logits of keys jt + lane and jt + 64 + lane
            float s[2];
            for (bool again = false;; again = true) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float v = 0.f;
                    if constexpr (BITS == 4) {
#pragma unroll
                        for (int w = NS - 1; w >= 0; --w) {
                            f32x4_t d = {0.f, 0.f, 0.f, 0.f};
                            if constexpr (DH == 32) d = mma_codes(qa[w], cur.k[u][0], d);
                            else {
                                d = mma_codes(qa[w], cur.k[2 * u][0], d);
                                d = mma_codes(qb[w], cur.k[2 * u + 1][0], d);
                            }
                            v = fmaf(v, 0x1p-20f, join_digits(d));
                        }
                    } else {
                        f32x4_t d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int w = 0; w < 4; ++w) {             // 8 codes of every lane's 32
                            const int p = w >> 1, e = 2 * (w & 1);
                            if constexpr (DH == 32) d = mma_bf16(ha[w], widen8(cur.k[u][p][e], cur.k[u][p][e + 1]), d);
                            else {
                                d = mma_bf16(ha[w], widen8(cur.k[2 * u][p][e], cur.k[2 * u][p][e + 1]), d);
                                d = mma_bf16(hb[w], widen8(cur.k[2 * u + 1][p][e], cur.k[2 * u + 1][p][e + 1]), d);
                            }
                        }
                        v = d[0];
#pragma unroll
                        for (int i = 1; i < NQ; ++i) v += d[i];
                    }
                    v *= bf16_bits(cur.ks[u]) * cq;
                    if constexpr (REL) v = fmaf(rel[hh * stretch + jt - c0 + 64 * u + lane], cs, v);
                    s[u] = cur.pad[u] ? -INFINITY : v;
                }
                if (!holes || again || !__builtin_amdgcn_ballot_w64(s[0] != s[0] || s[1] != s[1])) break;
#pragma unroll
                for (int w = 0; w < Tile<BITS, DH>::P; ++w)
#pragma unroll
                    for (int u = 0; u < Tile<BITS, DH>::NK; ++u) numbers(cur.k[u][w]);
            }
            // ---- running softmax
            const float mn = fmaxf(m, wave_max(fmaxf(s[0], s[1])));
            const float ms = mn == -INFINITY ? 0.f : mn;
            const float alpha = __builtin_amdgcn_exp2f(m - ms);
            m = mn;
            float p[2], x[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                p[u] = __builtin_amdgcn_exp2f(s[u] - ms);
                x[u] = cur.pad[u] ? 0.f : p[u] * bf16_bits(cur.vs[u]);      // a masked key's scale may be anything
            }
            lsum = fmaf(lsum, alpha, p[0] + p[1]);
            // ---- weights as operand rows 0 .. 3, then P V: lanes 0..15 get dimension 16 u + lane
            float f = 1.f, inv = 1.f;
            if constexpr (BITS == 4) {
                unit(wave_max(fmaxf(x[0], x[1])), f, inv);
                x[0] *= f;
                x[1] *= f;
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    const float d0 = rintf(x[0]), d1 = rintf(x[1]);
                    const int pk = __builtin_amdgcn_cvt_pk_fp8_f32(d0, d1, 0, false);
                    pw[i * PR + lane] = (uint8_t)pk;
                    pw[i * PR + 64 + lane] = (uint8_t)(pk >> 8);
                    x[0] = (x[0] - d0) * 32.f;
                    x[1] = (x[1] - d1) * 32.f;
                }
            } else {
#pragma unroll
                for (int i = 0; i < NP; ++i) {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const bf16_t d = (bf16_t)x[u];
                        reinterpret_cast<bf16_t*>(pw + i * PR)[64 * u + lane] = d;
                        x[u] -= (float)d;
                    }
                }
            }
            lds_order();
            if constexpr (BITS == 4) {
                i32x8_t pa[NS];
#pragma unroll
                for (int w = 0; w < NS; ++w) {
                    u32x4_t lo = zero, hi = zero;
                    if (c < 4 && 4 * w + c < NP) {
                        const uint8_t* pr = pw + (4 * w + c) * PR + 16 * g;
                        lo = *reinterpret_cast<const u32x4_t*>(pr);
                        hi = *reinterpret_cast<const u32x4_t*>(pr + 64);
                    }
                    pa[w] = two_pieces(lo, hi);
                }
                lds_order();
#pragma unroll
                for (int u = 0; u < DH / 16; ++u) {
                    float v = 0.f;
#pragma unroll
                    for (int w = NS - 1; w >= 0; --w) v = fmaf(v, 0x1p-20f, join_digits(mma_codes(pa[w], cur.v[u][0], (f32x4_t){0.f, 0.f, 0.f, 0.f})));
                    acc[u] = fmaf(acc[u], alpha, v * inv);
                }
            } else {
                bf16x8_t pa[4];                               // keys 8 w .. of every lane group's block
#pragma unroll
                for (int w = 0; w < 4; ++w)
                    pa[w] = __builtin_bit_cast(bf16x8_t, c < NP ? *reinterpret_cast<const u32x4_t*>(pw + c * PR + 64 * g + 16 * w) : zero);
                lds_order();
                float v[DH / 16];
                for (bool again = false;; again = true) {
                    bool none = false;
#pragma unroll
                    for (int u = 0; u < DH / 16; ++u) {
                        f32x4_t d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int w = 0; w < 4; ++w) d = mma_bf16(pa[w], widen8(cur.v[u][w >> 1][2 * (w & 1)], cur.v[u][w >> 1][2 * (w & 1) + 1]), d);
                        v[u] = d[0];
#pragma unroll
                        for (int i = 1; i < NP; ++i) v[u] += d[i];
                        none |= v[u] != v[u];
                    }
                    if (!holes || again || !__builtin_amdgcn_ballot_w64(none)) break;
#pragma unroll
                    for (int w = 0; w < Tile<BITS, DH>::P; ++w)
#pragma unroll
                        for (int u = 0; u < DH / 16; ++u) numbers(cur.v[u][w]);
                }
#pragma unroll
                for (int u = 0; u < DH / 16; ++u) acc[u] = fmaf(acc[u], alpha, v[u]);
            }
            if (more) cur = nxt;
        }
    }
    float l = wave_sum(lsum);
    if (kw > 1) {                                             // join the head's key ranges, in ascending order
        if (lane == 0) { jm[wid] = m; jl[wid] = l; }
#pragma unroll
        for (int u = 0; u < DH / 16; ++u) if (lane < 16) jo[wid][16 * u + lane] = acc[u];
        __syncthreads();
        if (wk != 0) return;
        for (int i = 1; i < kw; ++i) m = fmaxf(m, jm[wid + i]);
        const float ms = m == -INFINITY ? 0.f : m;
        l = 0.f;
#pragma unroll
        for (int u = 0; u < DH / 16; ++u) acc[u] = 0.f;
        for (int i = 0; i < kw; ++i) {
            const float w = __builtin_amdgcn_exp2f(jm[wid + i] - ms);
            l = fmaf(w, jl[wid + i], l);
#pragma unroll
            for (int u = 0; u < DH / 16; ++u) acc[u] = fmaf(w, jo[wid + i][16 * u + (lane & 15)], acc[u]);
        }
    }
    if (hw >= nh) return;
    if (a.part) {
        float* rec = a.part + (bh * a.nsplit + split) * ME_DEC_PART_REC(DH);
        if (lane == 0) *reinterpret_cast<f32x4_t*>(rec) = (f32x4_t){m * a.munit, l, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < DH / 16; ++u) if (lane < 16) rec[4 + 16 * u + lane] = acc[u];
    } else {
        T* o = reinterpret_cast<T*>(a.out) + (int64_t)b * a.sob + (int64_t)h * a.soh;
#pragma unroll
        for (int u = 0; u < DH / 16; ++u) if (lane < 16) o[16 * u + lane] = ET<T>::from_f(l == 0.f ? 0.f : acc[u] / l);
    }
}

// joins the key splits of a (sequence, head): one wave, splits in ascending order; no key left: zeros
template <typename T, int DH>
__global__ __launch_bounds__(256) void kvq_join_kernel(const float* __restrict__ part, int nsplit, int BH, int H, T* __restrict__ out, int64_t sob, int64_t soh) {
    const int lane = threadIdx.x & 63, bh = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (bh >= BH) return;
    constexpr int REC = ME_DEC_PART_REC(DH), U = 8;
    const float* rec = part + (size_t)bh * nsplit * REC;
    const float2 ml = lane < nsplit ? *reinterpret_cast<const float2*>(rec + (size_t)lane * REC) : make_float2(-INFINITY, 0.f);
    const float* po = rec + 4 + min(lane, DH - 1);
    float v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = po[(size_t)min(u, nsplit - 1) * REC];      // requested with the maxima: one round trip up to 8 splits
    const float mx = wave_max(ml.x), ms = mx == -INFINITY ? 0.f : mx;
    const float w = lane < nsplit ? exp2f(ml.x - ms) : 0.f, l = wave_sum(w * ml.y);
    float o = 0.f;
    for (int s0 = 0; s0 < nsplit; s0 += U) {
        float nx[U];
#pragma unroll
        for (int u = 0; u < U; ++u) nx[u] = s0 + U < nsplit ? po[(size_t)min(s0 + U + u, nsplit - 1) * REC] : 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float ws = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), min(s0 + u, 63)));
            if (s0 + u < nsplit) o = fmaf(ws, v[u], o);
            v[u] = nx[u];
        }
    }
    if (lane < DH) out[(int64_t)(bh / H) * sob + (int64_t)(bh % H) * soh + lane] = ET<T>::from_f(l == 0.f ? 0.f : o / l);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <typename T, int BITS, int DH> void launch_rows(bool write, bool vec, dim3 grid, hipStream_t st, const RowArgs& a) {
    if (write) {
        if (vec) kvq_write_kernel<T, BITS, DH, true><<<grid, 256, 0, st>>>(a);
        else kvq_write_kernel<T, BITS, DH, false><<<grid, 256, 0, st>>>(a);
    } else {
        if (vec) kvq_read_kernel<T, BITS, DH, true><<<grid, 256, 0, st>>>(a);
        else kvq_read_kernel<T, BITS, DH, false><<<grid, 256, 0, st>>>(a);
    }
}
template <typename T, int BITS> void launch_rows(bool write, bool vec, int dh, dim3 grid, hipStream_t st, const RowArgs& a) {
    if (dh == 32) launch_rows<T, BITS, 32>(write, vec, grid, st, a);
    else if (dh == 48) launch_rows<T, BITS, 48>(write, vec, grid, st, a);
    else launch_rows<T, BITS, 64>(write, vec, grid, st, a);
}

int cache_status(const me_kvq_cache* c) {
    if (!c || !c->kcodes || !c->kscale || !c->vcodes || !c->vscale) return ME_ERR_NULL;
    if ((c->dh != 32 && c->dh != 48 && c->dh != 64) || (c->bits != 4 && c->bits != 8) || c->B < 0 || c->H < 0 || c->blocks < 0 || c->blocks > (1 << 25) ||
        c->B > 65535 || c->H > 65535) return ME_ERR_BAD_SHAPE;
    return aligned16(c->kcodes) && aligned16(c->vcodes) ? ME_OK : ME_ERR_ALIGNMENT;
}

int rows_call(bool write, const me_kvq_cache* c, void* k, void* v, const int64_t* stride, int n, int t, const int32_t* t_dev, int ld_t,
              const int32_t* lens, int dtype, hipStream_t st) {
    me_clear_error();
    if (!k || !v || !stride) return ME_ERR_NULL;
    if (int rc = cache_status(c)) return rc;
    if (dtype != ME_F32 && dtype != ME_BF16 && dtype != ME_F16) return ME_ERR_BAD_DTYPE;
    if (n < 0 || (ld_t != 0 && ld_t != 1) || n > c->blocks * KB || (!t_dev && (t < 0 || (int64_t)t + n > (int64_t)c->blocks * KB))) return ME_ERR_BAD_SHAPE;
    if (c->B == 0 || n == 0 || c->H == 0) return ME_OK;
    const int es = dtype == ME_F32 ? 4 : 2;
    bool vec = aligned16(k) && aligned16(v);
    for (int i = 0; i < 6; ++i) vec = vec && (stride[i] * es) % 16 == 0;
    RowArgs a = {k, v, stride[0], stride[1], stride[2], stride[3], stride[4], stride[5], (uint8_t*)c->kcodes, (u16*)c->kscale, (uint8_t*)c->vcodes,
                 (u16*)c->vscale, n, c->H, c->blocks, t, ld_t, t_dev, lens};
    // blocks that n tokens from any position can touch (from t where it is known)
    const int nblk = t_dev ? (n + KB - 2) / KB + 1 : (t + n - 1) / KB - t / KB + 1;
    const dim3 grid(nblk, c->H, c->B);
#define ME_KVQ_ROWS(T) (c->bits == 4 ? launch_rows<T, 4>(write, vec, c->dh, grid, st, a) : launch_rows<T, 8>(write, vec, c->dh, grid, st, a))
    if (dtype == ME_F32) ME_KVQ_ROWS(float);
    else if (dtype == ME_BF16) ME_KVQ_ROWS(bf16_t);
    else ME_KVQ_ROWS(f16_t);
#undef ME_KVQ_ROWS
    return me_launch_status();
}

template <typename T, int BITS, int DH> void launch_attn(dim3 grid, int threads, hipStream_t st, const AttnArgs& a) {
    if (a.E) kvq_attn_kernel<T, BITS, DH, true><<<grid, threads, 0, st>>>(a);
    else kvq_attn_kernel<T, BITS, DH, false><<<grid, threads, 0, st>>>(a);
}
template <typename T> void attn_call(const AttnArgs& a, int B, int dh, int bits, bool join, hipStream_t st) {
    const dim3 grid(a.nsplit, (a.H + a.hpb - 1) / a.hpb, B);
    const int threads = 64 * a.hpb * a.kw;
#define ME_KVQ_ATTN(DHV) (bits == 4 ? launch_attn<T, 4, DHV>(grid, threads, st, a) : launch_attn<T, 8, DHV>(grid, threads, st, a))
    if (dh == 32) ME_KVQ_ATTN(32); else if (dh == 48) ME_KVQ_ATTN(48); else ME_KVQ_ATTN(64);
#undef ME_KVQ_ATTN
    if (!join) return;
    const int BH = B * a.H;
    T* out = reinterpret_cast<T*>(a.out);
    if (dh == 32) kvq_join_kernel<T, 32><<<(BH + 3) / 4, 256, 0, st>>>(a.part, a.nsplit, BH, a.H, out, a.sob, a.soh);
    else if (dh == 48) kvq_join_kernel<T, 48><<<(BH + 3) / 4, 256, 0, st>>>(a.part, a.nsplit, BH, a.H, out, a.sob, a.soh);
    else kvq_join_kernel<T, 64><<<(BH + 3) / 4, 256, 0, st>>>(a.part, a.nsplit, BH, a.H, out, a.sob, a.soh);
}

}  // namespace

extern "C" {

int me_kvq_write(const me_kvq_cache* c, const void* k, const void* v, const int64_t* strides, int n, int t, const int32_t* t_dev, int ld_t,
                 const int32_t* lens, int dtype, void* stream) {
    return rows_call(true, c, const_cast<void*>(k), const_cast<void*>(v), strides, n, t, t_dev, ld_t, lens, dtype, (hipStream_t)stream);
}

int me_kvq_read(const me_kvq_cache* c, void* k, void* v, const int64_t* strides, int n, int t, const int32_t* t_dev, int ld_t, const int32_t* lens,
                int dtype, void* stream) {
    return rows_call(false, c, k, v, strides, n, t, t_dev, ld_t, lens, dtype, (hipStream_t)stream);
}

// How the keys are cut.  2048 waves (8 per CU) are enough to keep the memory busy; a row (sequence, head) that has fewer is cut into
// ranges: first inside the block (ranges meet in LDS), then over blocks, whose records a second launch joins (2 .. 3 us).  The
// relative products want blocks of many heads (a stretch's rows of E are read once per block) but 256 blocks, one per CU, come first.
// Measured, us per call of one cache replayed (it stays in the last-level cache), 4 bits, dh 64, one block per row and all ranges in it -> as chosen here:
//   relative table: 1 x 8 rows of 2048 keys 13.5 -> 7.4, 4 x 8: 14.5 -> 8.0, 16 x 8: 15.6 -> 11.2, 64 x 8: 34.0 -> 20.4; up to 512 keys
//   one launch is faster (4 x 8 of 512: 6.5, four splits 7.0);  none: 1 x 8 of 16384 keys 8 splits 9.2, 16: 8.5; 16 x 8 of 4096: two splits 12.6, none 12.0.
int me_kvq_splits(int B, int H, int tokens, int rel) {
    if (B <= 0 || H <= 0 || tokens <= 0) return 1;
    const int64_t rows = (int64_t)B * H, tiles = ((int64_t)tokens + TK - 1) / TK;
    if (rel) return tiles <= 4 || rows > 512 ? 1 : (int)std::min<int64_t>(std::min<int64_t>(2048 / rows, tiles), 64);
    const int64_t ns = std::min<int64_t>(std::min<int64_t>(2048 / (rows * WAVES), tiles / WAVES), 64);
    return ns > 2 ? (int)ns : 1;
}

static int attn_entry(const me_kvq_cache* c, const void* q, int64_t ldq_b, int64_t ldq_h, const void* kn, const void* vn, int64_t ldn_b, int64_t ldn_h,
                      const void* E, int M, const uint8_t* key_pad, int ld_pad, void* out, int64_t ldo_b, int64_t ldo_h, float* part, size_t part_bytes,
                      int nsplit, int t, const int32_t* t_dev, int ld_t, int dtype, void* stream) {
    me_clear_error();
    if (!q || (!out && !part)) return ME_ERR_NULL;
    if (int rc = cache_status(c)) return rc;
    if (dtype != ME_F32 && dtype != ME_BF16 && dtype != ME_F16) return ME_ERR_BAD_DTYPE;
    if (nsplit < 1 || nsplit > 64 || (ld_t != 0 && ld_t != 1) || (!t_dev && (t < -1 || t >= c->blocks * KB)) || (E && M < c->blocks * KB) ||
        (key_pad && ld_pad < 0)) return ME_ERR_BAD_SHAPE;
    const int es = dtype == ME_F32 ? 4 : 2;
    if ((E && !aligned16(E)) || (part && !aligned16(part)) || (kn && (!aligned16(kn) || !aligned16(vn) || (ldn_b * es) % 16 || (ldn_h * es) % 16))) return ME_ERR_ALIGNMENT;
    if (c->B == 0 || c->H == 0) return ME_OK;
    const bool split = nsplit > 1 || !out;                    // out == NULL: the partial records are the result (me_dec_proj_resid joins them)
    if (split && (!part || part_bytes < (size_t)c->B * c->H * nsplit * ME_DEC_PART_REC(c->dh) * 4)) return ME_ERR_WORKSPACE;
    // key ranges inside the block up to 2048 waves, then heads into the block while 256 blocks are left (see me_kvq_splits)
    int hpb = 1, kw = 1;
    const int64_t tiles = ((((t_dev ? (int64_t)c->blocks * KB : (int64_t)t + 1) + nsplit - 1) / nsplit) + TK - 1) / TK, cut = (int64_t)nsplit * c->B;
    while (kw < WAVES && kw < tiles && cut * c->H * kw <= 1024) kw *= 2;
    while (E && hpb * kw < WAVES && hpb < HG && 2 * hpb <= c->H && cut * ((c->H + 2 * hpb - 1) / (2 * hpb)) >= 256) hpb *= 2;
    AttnArgs a = {q, ldq_b, ldq_h, (const uint8_t*)c->kcodes, (const u16*)c->kscale, (const uint8_t*)c->vcodes, (const u16*)c->vscale, E, M, key_pad, ld_pad,
                  out, ldo_b, ldo_h, split ? part : nullptr, nsplit, kn, vn, ldn_b, ldn_h, c->H, c->blocks, t, ld_t, hpb, kw, t_dev, 1.f / sqrtf((float)c->dh), out ? 1.f : 0.6931471805599453f};
    if (dtype == ME_F32) attn_call<float>(a, c->B, c->dh, c->bits, split && out, (hipStream_t)stream);
    else if (dtype == ME_BF16) attn_call<bf16_t>(a, c->B, c->dh, c->bits, split && out, (hipStream_t)stream);
    else attn_call<f16_t>(a, c->B, c->dh, c->bits, split && out, (hipStream_t)stream);
    return me_launch_status();
}

int me_kvq_attn(const me_kvq_cache* c, const void* q, int64_t ldq_b, int64_t ldq_h, const void* E, int M, const uint8_t* key_pad, int ld_pad,
                void* out, int64_t ldo_b, int64_t ldo_h, float* part, size_t part_bytes, int nsplit, int t, const int32_t* t_dev, int ld_t, int dtype,
                void* stream) {
    return attn_entry(c, q, ldq_b, ldq_h, nullptr, nullptr, 0, 0, E, M, key_pad, ld_pad, out, ldo_b, ldo_h, part, part_bytes, nsplit, t, t_dev, ld_t, dtype, stream);
}

int me_kvq_append_attn(const me_kvq_cache* c, const void* q, int64_t ldq_b, int64_t ldq_h, const void* k, const void* v, int64_t ldn_b, int64_t ldn_h,
                       const void* E, int M, const uint8_t* key_pad, int ld_pad, void* out, int64_t ldo_b, int64_t ldo_h, float* part, size_t part_bytes,
                       int nsplit, int t, const int32_t* t_dev, int ld_t, int dtype, void* stream) {
    if (!k || !v) return ME_ERR_NULL;
    if (!t_dev && t < 0) return ME_ERR_BAD_SHAPE;
    return attn_entry(c, q, ldq_b, ldq_h, k, v, ldn_b, ldn_h, E, M, key_pad, ld_pad, out, ldo_b, ldo_h, part, part_bytes, nsplit, t, t_dev, ld_t, dtype, stream);
}

}  // extern "C"
