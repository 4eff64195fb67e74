// KV cache by handle (include/seedmi.h: seedmi_kv_cache_t): rows written, read back and attended to.
//
//  seedmi_kv_append     apply_rotary_pos_emb + append (llama_xformer.py:160-168, 234-239) into 16-bit or 8-bit rows, grouped heads, one
//                       length per slot
//  seedmi_kv_read       8-bit rows back as 16-bit tensors
//  seedmi_kv_attention  memory_efficient_attention over the cache (llama_xformer.py:244-256), optionally behind a prefix that all slots share
#include <float.h>
#include <limits.h>
#include <math.h>
#include <string.h>
#include "common.h"
#include "seedmi_internal.h"
#include "../../include/seedmi.h"

namespace {

// ------------------------------------------------------------------------------------------------ the 8-bit block format
// e4m3 has 3 mantissa bits whatever its exponent, so a power-of-two scale costs no precision against a free one; it makes both directions
// exact apart from the one rounding (x * 2^-e and code * 2^e are exact), and it is what the conversion instructions take.
#ifdef SEEDMI_F16
constexpr float MX_TOP = 61440.f;                       // 1.875 * 2^15: the largest e4m3-grid value that is finite in the element type
#else
constexpr float MX_TOP = 0x1.ep127f;                    // 1.875 * 2^127
#endif

SEEDMI_DEVINL bool is_finite_f(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }
// magnitude that enters a block's maximum
SEEDMI_DEVINL float mx_mag(float x) { return is_finite_f(x) ? fminf(fabsf(x), MX_TOP) : 0.f; }
// scale byte of a block whose largest magnitude is a: biased exponent of a, + 1 if its mantissa is above 1.75 (the carry), - 8
SEEDMI_DEVINL unsigned mx_scale_byte(float a) {
    const int b = (int)((__float_as_uint(a) + 0x1fffffu) >> 23) - 8;
    return (unsigned)max(b, 1);
}
// value handed to the e4m3 conversion: exact, |.| <= 448
SEEDMI_DEVINL float mx_scaled(float x, unsigned byte) {
    const float inv = __uint_as_float((254u - byte) << 23);
    return is_finite_f(x) ? fminf(fmaxf(x, -MX_TOP), MX_TOP) * inv : __uint_as_float(0x7fc00000u);
}
SEEDMI_DEVINL unsigned mx_pack4(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
// two e4m3 bytes (low / high half of w) times 2^(byte - 127) as two 16-bit elements; `scale` = the float with that exponent
template <bool HI>
SEEDMI_DEVINL uint32_t mx_unpack2(uint32_t w, float scale) {
#ifdef SEEDMI_F16
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI));
#else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
#endif
}
SEEDMI_DEVINL float mx_scale_f(unsigned byte) { return __uint_as_float(byte << 23); }

struct KvView {                                          // seedmi_kv_cache_t as the kernels take it
    char *k, *v;
    uint8_t *ks, *vs;
    long long slot_rows, head_rows;
    int rows, G;
};

// ------------------------------------------------------------------------------------------------ append
// y = half(half(x cos) + half(rotate_half(x) sin)); per block of 32 y: a = max |y|, e = min {e : a <= 448 2^e}, codes e4m3(y 2^-e).
// One thread = 8 values i .. i + 7 and their partners i + HD/2 .. of one (slot, token, head): a quad of lanes holds two whole blocks of 32,
// and the block maximum is two exchanges.  Bound by its bytes: 8 x 649 tokens of 40 heads (268 MB) take 59 us, 4.5 TB/s; a step of one or
// 32 tokens 3 - 5 us, which is a launch.
template <int HD, bool MX>
__global__ __launch_bounds__(256) void kv_append_kernel(const KvView c, const bf16_t* __restrict__ qkv, int ldqkv,
                                                        const long long* __restrict__ pos_ids, int pos_base,
                                                        const bf16_t* __restrict__ cos_t, const bf16_t* __restrict__ sin_t, int max_pos,
                                                        bf16_t* __restrict__ q_out, int ldq, int B, int T, int H, int past_len,
                                                        const int* __restrict__ past_lens) {
    constexpr int LPR = HD / 16;                         // lanes per head row
    const int heads = H + 2 * c.G;
    const unsigned idx = blockIdx.x * 256u + threadIdx.x;
    const unsigned total = (unsigned)B * T * heads * LPR;
    if (idx >= total) return;                            // (whole quads: total is a multiple of 4)
    const int l = idx % LPR;
    const unsigned r = idx / LPR;
    const int h = r % heads;
    const unsigned row = r / heads;
    const int b = row / T, t = row - b * T;
    const int past = past_lens ? past_lens[b] : past_len;
    const bf16_t* src = qkv + (size_t)row * ldqkv + h * HD;
    const int i0 = 8 * l;
    const uint4 a = *(const uint4*)(src + i0), z = *(const uint4*)(src + i0 + HD / 2);
    const unsigned aw[4] = {a.x, a.y, a.z, a.w}, zw[4] = {z.x, z.y, z.z, z.w};
    float x1[8], x2[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        x1[2 * j] = lo_bf(aw[j]); x1[2 * j + 1] = hi_bf(aw[j]);
        x2[2 * j] = lo_bf(zw[j]); x2[2 * j + 1] = hi_bf(zw[j]);
    }
    if (h < H + c.G) {                                   // half(half(x cos) + half(rotate_half(x) sin)), llama_xformer.py:160-168
#pragma clang fp contract(off)                           // (fp16: a fused multiply-add would leave out the rounding of one product)
        long long pos = pos_ids ? pos_ids[row] : (long long)pos_base + past + t;
        pos = pos < 0 ? 0 : (pos >= max_pos ? max_pos - 1 : pos);
        const bf16_t* cs = cos_t + pos * HD;
        const bf16_t* sn = sin_t + pos * HD;
        const uint4 c1 = *(const uint4*)(cs + i0), c2 = *(const uint4*)(cs + i0 + HD / 2);
        const uint4 s1 = *(const uint4*)(sn + i0), s2 = *(const uint4*)(sn + i0 + HD / 2);
        const unsigned c1w[4] = {c1.x, c1.y, c1.z, c1.w}, c2w[4] = {c2.x, c2.y, c2.z, c2.w};
        const unsigned s1w[4] = {s1.x, s1.y, s1.z, s1.w}, s2w[4] = {s2.x, s2.y, s2.z, s2.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float u = x1[j], w = x2[j];
            const float C1 = j & 1 ? hi_bf(c1w[j >> 1]) : lo_bf(c1w[j >> 1]), S1 = j & 1 ? hi_bf(s1w[j >> 1]) : lo_bf(s1w[j >> 1]);
            const float C2 = j & 1 ? hi_bf(c2w[j >> 1]) : lo_bf(c2w[j >> 1]), S2 = j & 1 ? hi_bf(s2w[j >> 1]) : lo_bf(s2w[j >> 1]);
            x1[j] = rbf(rbf(u * C1) + rbf(-w * S1));
            x2[j] = rbf(rbf(w * C2) + rbf(u * S2));
        }
    }
    const uint4 o1 = make_uint4(pack2bf(x1[0], x1[1]), pack2bf(x1[2], x1[3]), pack2bf(x1[4], x1[5]), pack2bf(x1[6], x1[7]));
    const uint4 o2 = make_uint4(pack2bf(x2[0], x2[1]), pack2bf(x2[2], x2[3]), pack2bf(x2[4], x2[5]), pack2bf(x2[6], x2[7]));
    // largest magnitudes of the quad's two blocks (every lane of the wave takes part, whatever its row is)
    float m1 = 0.f, m2 = 0.f;
    if (MX) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            m1 = fmaxf(m1, mx_mag(x1[j]));
            m2 = fmaxf(m2, mx_mag(x2[j]));
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            m1 = fmaxf(m1, __shfl_xor(m1, o, 64));
            m2 = fmaxf(m2, __shfl_xor(m2, o, 64));
        }
    }
    if (h < H) {
        bf16_t* qo = q_out + (size_t)row * ldq + h * HD + i0;
        *(uint4*)qo = o1;
        *(uint4*)(qo + HD / 2) = o2;
        return;
    }
    const long long at = (long long)past + t;
    if (past < 0 || at >= c.rows) return;                // idle slot / a row beyond the cache
    const bool is_v = h >= H + c.G;
    const int g = h - H - (is_v ? c.G : 0);
    const long long crow = (long long)b * c.slot_rows + (long long)g * c.head_rows + at;
    if (MX) {
        const unsigned b1 = mx_scale_byte(m1), b2 = mx_scale_byte(m2);
        float y1[8], y2[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) { y1[j] = mx_scaled(x1[j], b1); y2[j] = mx_scaled(x2[j], b2); }
        char* dst = (is_v ? c.v : c.k) + crow * HD + i0;
        *(uint2*)dst = make_uint2(mx_pack4(y1[0], y1[1], y1[2], y1[3]), mx_pack4(y1[4], y1[5], y1[6], y1[7]));
        *(uint2*)(dst + HD / 2) = make_uint2(mx_pack4(y2[0], y2[1], y2[2], y2[3]), mx_pack4(y2[4], y2[5], y2[6], y2[7]));
        if ((l & 3) == 0) {
            uint8_t* sc = (is_v ? c.vs : c.ks) + crow * (HD / 32) + (l >> 2);
            sc[0] = (uint8_t)b1;
            sc[HD / 64] = (uint8_t)b2;
        }
    } else {
        bf16_t* dst = (bf16_t*)(is_v ? c.v : c.k) + crow * HD + i0;
        *(uint4*)dst = o1;
        *(uint4*)(dst + HD / 2) = o2;
    }
}

// ------------------------------------------------------------------------------------------------ read back
// One thread = 16 values: 16 code bytes in, 32 bytes out.  blockIdx.y: keys / values.  Bound by its bytes: 4 x 8191 rows of 32 heads (814 MB)
// take 133 us, 6.1 TB/s (a copy of a gigabyte reaches 5.1 on this card, a read-only stream 7.0).
template <int HD>
__global__ __launch_bounds__(256) void kv_read_kernel(const KvView c, bf16_t* __restrict__ k_out, bf16_t* __restrict__ v_out, int B, int n,
                                                      int start, const int* __restrict__ starts) {
    constexpr int LPR = HD / 16;
    const bool is_v = k_out == nullptr || blockIdx.y == 1;
    const long long total = (long long)B * c.G * n * LPR;
    for (long long idx = (long long)blockIdx.x * 256 + threadIdx.x; idx < total; idx += (long long)gridDim.x * 256) {
        const int l = (int)(idx % LPR);
        const long long r = idx / LPR;                   // output row
        const int i = (int)(r % n);
        const int bg = (int)(r / n);
        const int b = bg / c.G, g = bg - b * c.G;
        const long long at = (long long)(starts ? starts[b] : start) + i;
        uint4* dst = (uint4*)((is_v ? v_out : k_out) + r * HD + 16 * l);
        if (at < 0 || at >= c.rows) {
            dst[0] = dst[1] = make_uint4(0, 0, 0, 0);
            continue;
        }
        const long long crow = (long long)b * c.slot_rows + (long long)g * c.head_rows + at;
        const uint4 w = *(const uint4*)((is_v ? c.v : c.k) + crow * HD + 16 * l);
        const float s = mx_scale_f(((is_v ? c.vs : c.ks) + crow * (HD / 32))[l >> 1]);
        dst[0] = make_uint4(mx_unpack2<false>(w.x, s), mx_unpack2<true>(w.x, s), mx_unpack2<false>(w.y, s), mx_unpack2<true>(w.y, s));
        dst[1] = make_uint4(mx_unpack2<false>(w.z, s), mx_unpack2<true>(w.z, s), mx_unpack2<false>(w.w, s), mx_unpack2<true>(w.w, s));
    }
}

// ------------------------------------------------------------------------------------------------ attention
// Query rows that read the same keys form a GROUP: the T * (H / G) rows of a (slot, key head) over the slot's own rows, or all
// B * T * (H / G) rows of a key head over the shared prefix.  Row r of a group is token row base + r / GH (GH = H / G), head g * GH + r % GH.
//
// With s_j = c q.k_j (c = scale * log2 e) a range of keys gives m = reference(max s_j), l = sum 2^(s_j - m), o = sum 2^(s_j - m) v_j; ranges
// join by M = max m, (l, o) = sum 2^(m - M) (l, o), and out = o / l.
struct AttnPass {                                       // one pass: the slots' own rows, or the shared prefix
    KvView c;                                            // the slots' cache, or the prefix as a cache of one slot
    const int* kv_lens;
    int kv_len, shared;                                  // shared: the groups are those of the prefix (kv_len rows, all visible)
    int groups, group_rows, row_blocks;                  // groups = slots * G (prefix: G), rows of a group, row blocks of a group
    int splits, part0, per_split;                        // key ranges, the first one's part index, tiles of a range (at least)
    unsigned blocks;                                     // workgroups of the pass
};
struct AttnArgs {
    const bf16_t* q;
    bf16_t* out;
    float* o_part;                                       // [parts][B*T*H][HD] sums of a part; parts == 1: unused, results go to out
    float2* ml_part;                                     // [parts][B*T*H] (m, l); l == 0: the part holds nothing for the row
    unsigned* arrivals;                                  // one counter per unit that is joined (join_in_place), else NULL
    int ldq, ldo, T, H, GH, causal, parts;
    unsigned unit_blocks;                                // workgroups that arrive at a unit's counter
    int unit_rows;                                       // rows of a unit where it is a whole key head (two passes), else 0
    long long rows;                                      // B * T * H
    float c2;
    AttnPass pass[2];
};
// The pass a workgroup belongs to, field by field (scalar selects; an indexed kernel argument would be copied to memory).
SEEDMI_DEVINL AttnPass pass_of(const AttnArgs& a, unsigned& block) {
    const bool second = blockIdx.x >= a.pass[0].blocks;
    block = blockIdx.x - (second ? a.pass[0].blocks : 0u);
    AttnPass p;
#define SEL(f) p.f = second ? a.pass[1].f : a.pass[0].f
    SEL(c.k); SEL(c.v); SEL(c.ks); SEL(c.vs); SEL(c.slot_rows); SEL(c.head_rows); SEL(c.rows); SEL(c.G);
    SEL(kv_lens); SEL(kv_len); SEL(shared); SEL(groups); SEL(group_rows); SEL(row_blocks); SEL(splits); SEL(part0); SEL(per_split); SEL(blocks);
#undef SEL
    return p;
}

// rows of a pass's slot that count: kv_len, on top of what the slot's own length says where there is one (negative: an idle slot), within the cache
SEEDMI_DEVINL int rows_of_slot(const int* kv_lens, int kv_len, int rows, int slot) {
    int n = kv_len;
    if (kv_lens) {
        const int own = kv_lens[slot];
        n = own < 0 ? 0 : min(own, rows) + n;
    }
    return max(0, min(n, rows));
}
SEEDMI_DEVINL int rows_held(const AttnPass& p, int slot) {
    return __builtin_amdgcn_readfirstlane(rows_of_slot(p.shared ? nullptr : p.kv_lens, p.kv_len, p.c.rows, slot));
}

typedef __attribute__((ext_vector_type(4))) short s16x4;
constexpr int KT = 32;                                   // keys of a tile
constexpr int MIN_TILES = 4;                             // of a split: one tile per wave

// maximum of three that a NaN goes through (v_maximum3_f32; fmaxf would quieten each of its operands first: three instructions for one)
SEEDMI_DEVINL float max3(float a, float b, float c) { return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c); }
SEEDMI_DEVINL float max2(float a, float b) { return __builtin_elementwise_maximum(a, b); }
// maximum / sum over the four 16-lane rows of a wave (the lanes of one query): VALU row swaps, no LDS
SEEDMI_DEVINL float rows_max(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = max2(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return max2(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
SEEDMI_DEVINL float rows_sum(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
SEEDMI_DEVINL float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
// acc + lo + hi of a word of two 16-bit elements: a dot product with ones
SEEDMI_DEVINL float add_pair(uint32_t w, float acc) {
#ifdef SEEDMI_F16
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(hw_f16x2, w), __builtin_bit_cast(hw_f16x2, 0x3c003c00u), acc, false);
#else
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(hw_bf16x2, w), __builtin_bit_cast(hw_bf16x2, 0x3f803f80u), acc, false);
#endif
}
// Probabilities are rounded to the element for the product with the values, whose matrix instructions take operands of one type: in bf16 the
// error against 64 bits is 0.0017 - 0.0019 relative, 0.0016 - 0.0018 of it the output's own rounding (fp16: 0.00022, 0.00021).  The sum of a
// row is that of its probabilities as they are rounded: out is then a mean of the values with weights that add up to one, in every kernel.
// (A sum of unrounded ones is off by what the roundings have in common: 387 equal scores of 400 made every output 0.92 half steps too small.)
SEEDMI_DEVINL float add_probabilities(const uint4& w, float acc) { return add_pair(w.w, add_pair(w.z, add_pair(w.y, add_pair(w.x, acc)))); }

// a product that is rounded before it is used (the compiler would be free to fuse it)
SEEDMI_DEVINL float rounded(float x) {
    asm("" : "+v"(x));
    return x;
}
// What a row's exponents are taken against, given its largest score so far (in base-2 exponents): a probability leaves as 2^(score - reference),
// rounded to the element.  bf16: the largest score, probabilities <= 1.  fp16 ends at 2^-25, far above what many thousand keys may add up from:
// 15 less, so that probabilities reach from 2^15 down to 2^-25, 2^-40 of the largest.  Sums and values have the factor in common.
// FAR: from there on score and reference are rounded by more than a sixteenth before they are subtracted, and the fused s c - reference of the
// largest score, the rounding of s c, would no longer be near zero (2^32 and more: a probability of 2^128 or of 0).  A wave with a reference
// beyond it rounds s c like the reference, so that the largest score's exponent is exactly 0, and takes no 15 off.
constexpr float FAR = 0x1p20f;
SEEDMI_DEVINL float reference(float m) {
#ifdef SEEDMI_F16
    return m == -INFINITY ? 0.f : fabsf(m) < FAR ? m - 15.f : m;
#else
    return m == -INFINITY ? 0.f : m;
#endif
}

// not finite: exponent field all ones, in both halves of a word of 16-bit elements
SEEDMI_DEVINL uint32_t exp_mask16() {
#ifdef SEEDMI_F16
    return 0x7c00u;
#else
    return 0x7f80u;
#endif
}
SEEDMI_DEVINL bool bad16(uint32_t h) { return (h & exp_mask16()) == exp_mask16(); }
SEEDMI_DEVINL bool bad_word(uint32_t w) { return bad16(w) | bad16(w >> 16); }
SEEDMI_DEVINL bool bad_words(const uint4& w) { return bad_word(w.x) | bad_word(w.y) | bad_word(w.z) | bad_word(w.w); }
// zeros in place of what is not finite
SEEDMI_DEVINL uint32_t clean_word(uint32_t w) { return (bad16(w) ? 0u : w & 0xffffu) | (bad16(w >> 16) ? 0u : w & 0xffff0000u); }

// The rows 0 .. n - 1 of a (slot, head) as buffers: a load takes a per-lane offset that never changes and a scalar one for the tile, and
// rows from n on read as zeros without touching memory.  (The scalar offset counts in the range check, a load whose scalar offset alone is at
// or beyond the end included - the requests for a tile behind the last one: tools/probes/buffer_range_probe.hip, every size of load.)
struct RowBuffers { __amdgpu_buffer_rsrc_t k, v, ks, vs; };
template <int HD, bool MX>
SEEDMI_DEVINL RowBuffers row_buffers(const KvView& c, long long row0, int n) {
    constexpr int RB = MX ? HD : 2 * HD;
    RowBuffers b;
    b.k = __builtin_amdgcn_make_buffer_rsrc(c.k + row0 * RB, 0, n * RB, 0x00020000);
    b.v = __builtin_amdgcn_make_buffer_rsrc(c.v + row0 * RB, 0, n * RB, 0x00020000);
    b.ks = __builtin_amdgcn_make_buffer_rsrc(MX ? c.ks + row0 * (HD / 32) : (uint8_t*)c.k, 0, MX ? n * (HD / 32) : 0, 0x00020000);
    b.vs = __builtin_amdgcn_make_buffer_rsrc(MX ? c.vs + row0 * (HD / 32) : (uint8_t*)c.k, 0, MX ? n * (HD / 32) : 0, 0x00020000);
    return b;
}
SEEDMI_DEVINL uint4 load16(const __amdgpu_buffer_rsrc_t& r, int lane_off, int tile_off) {
    const seedmi_u32x4 w = __builtin_amdgcn_raw_buffer_load_b128(r, lane_off, tile_off, 0);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Scale bytes of a row, for a lane that needs the one of block `blk`.  Rows of 128 values: the row's four bytes as one word, the byte taken at
// its use.  (A byte load is widened in the loop's last block by this compiler: a wait for the loads of the next tile, in every iteration.
// Rows of 64 have two bytes and no word of their own.)
template <int HD>
SEEDMI_DEVINL uint32_t load_scale(const __amdgpu_buffer_rsrc_t& r, int row, int blk, int tile_off) {
    if (HD == 128) return __builtin_amdgcn_raw_buffer_load_b32(r, row * 4, tile_off, 0);
    return __builtin_amdgcn_raw_buffer_load_b8(r, row * (HD / 32) + blk, tile_off, 0);
}
template <int HD>
SEEDMI_DEVINL float scale_of(uint32_t loaded, int blk) { return mx_scale_f(HD == 128 ? (loaded >> (8 * blk)) & 255u : loaded); }

// A tile of 32 keys and values as a wave holds it between the load and its use.
//   K (the MFMA's A operand, rows = keys): lane (li, g) holds its part of rows 16 kt + li.  16-bit rows: k-step ks = values 32 ks + 8 g ..;
//     8-bit rows: 16 bytes at 64 j + 16 g = k-steps 2 j and 2 j + 1 (the contraction may run in any order that Q's fragments share).
//   V: whole rows, lanes side by side.
template <int HD, bool MX>
struct Tile {
    static constexpr int KL = MX ? HD / 64 : HD / 32;    // 16-byte loads of a key row per lane
    static constexpr int VL = MX ? HD / 32 : HD / 16;    // 16-byte loads of the value tile per lane
    uint4 k[2][KL], v[VL];
    uint32_t ks[2], vs[VL];
};

template <int HD, bool MX>
SEEDMI_DEVINL void load_k(Tile<HD, MX>& t, const RowBuffers& b, int key0, int lane) {
    constexpr int RB = MX ? HD : 2 * HD;                 // bytes of a row
    const int li = lane & 15, g = lane >> 4;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
        for (int j = 0; j < Tile<HD, MX>::KL; ++j) t.k[kt][j] = load16(b.k, li * RB + 16 * g + 16 * kt * RB + 64 * j, key0 * RB);
        if (MX) t.ks[kt] = HD == 128 ? __builtin_amdgcn_raw_buffer_load_b32(b.ks, li * 4 + 64 * kt, key0 * 4, 0)
                                     : (uint32_t)__builtin_amdgcn_raw_buffer_load_b16(b.ks, li * 2 + 32 * kt, key0 * 2, 0);
    }
}
template <int HD, bool MX>
SEEDMI_DEVINL void load_v(Tile<HD, MX>& t, const RowBuffers& b, int key0, int lane) {
    constexpr int RB = MX ? HD : 2 * HD;
    constexpr int LPR = RB / 16;                         // lanes of a row
#pragma unroll
    for (int j = 0; j < Tile<HD, MX>::VL; ++j) {
        t.v[j] = load16(b.v, lane * 16 + 1024 * j, key0 * RB);
        if (MX) t.vs[j] = load_scale<HD>(b.vs, lane / LPR + j * (64 / LPR), (lane % LPR) / 2, key0 * (HD / 32));
    }
}

// LDS images of widened tiles: rows of 2 HD bytes, padded so that the rows that are read together lie on different banks (keys: 16 bytes of
// 16 rows at a time; values: 32 bytes of 8 rows, the transposing read) and every address is a lane's own plus a constant.
template <int HD>
SEEDMI_DEVINL constexpr int k_at(int row, int c) { return row * (2 * HD + 16) + 16 * c; }                // 16-byte chunk c of a key row
template <int HD>
SEEDMI_DEVINL constexpr int v_at(int row, int c) { return row * (2 * HD + 32) + 16 * c; }                // ... of a value row

// The value tile into the LDS image.  LOOK: returns whether this lane saw a value that is not finite.
template <int HD, bool MX, bool LOOK>
SEEDMI_DEVINL bool stage_v(const Tile<HD, MX>& t, char* lds, int lane) {
    constexpr int LPR = (MX ? HD : 2 * HD) / 16;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < Tile<HD, MX>::VL; ++j) {
        const int row = j * (64 / LPR) + lane / LPR, l = lane % LPR;
        const uint4 w = t.v[j];
        const uint32_t src[4] = {w.x, w.y, w.z, w.w};
        if (MX) {
            const float s = scale_of<HD>(t.vs[j], l / 2);
            uint32_t o[8];
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                o[2 * d] = mx_unpack2<false>(src[d], s);
                o[2 * d + 1] = mx_unpack2<true>(src[d], s);
                if (LOOK) bad |= bad_word(o[2 * d]) | bad_word(o[2 * d + 1]);
            }
            *(uint4*)(lds + v_at<HD>(row, 2 * l)) = make_uint4(o[0], o[1], o[2], o[3]);
            *(uint4*)(lds + v_at<HD>(row, 2 * l + 1)) = make_uint4(o[4], o[5], o[6], o[7]);
        } else {
#pragma unroll
            for (int d = 0; d < 4; ++d)
                if (LOOK) bad |= bad_word(src[d]);
            *(uint4*)(lds + v_at<HD>(row, l)) = w;
        }
    }
    return bad;
}

// V^T fragment of channels 16 n .. + 15 from the LDS image: lane li = channel, keys 16 (j >> 2) + 4 g + (j & 3)
template <int HD>
SEEDMI_DEVINL bf16x8 v_frag(const char* lds, int n, int lane) {
    const int li = lane & 15, g = lane >> 4;
    const int row = 4 * g + (li >> 2), c = 2 * n + ((li & 3) >> 1), b8 = (li & 1) << 3;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds + v_at<HD>(row, c) + b8));
    const s16x4 z = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds + v_at<HD>(row + 16, c) + b8));
    const uint2 lo = __builtin_bit_cast(uint2, a), hi = __builtin_bit_cast(uint2, z);
    return __builtin_bit_cast(bf16x8, make_uint4(lo.x, lo.y, hi.x, hi.y));
}

// The values are used here: the wait for their loads ends before a loop, whose own waits then count only the loads of its tiles (a wait that
// also covers these would be a wait for everything in flight, in every iteration).
template <int N, int M>
SEEDMI_DEVINL void arrived(bf16x8 (&x)[N][M]) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < M; ++j) asm volatile("" : "+v"(x[i][j]));
}
constexpr float LOWEST = -3.4028234e38f;
SEEDMI_DEVINL void lds_fence() { asm volatile("" ::: "memory"); }        // (a wave's own LDS accesses are executed in order)

// ---- joining the parts of a row
// (m, l, o) of a running join with one more part.  M starts at LOWEST, L and o at zero.
SEEDMI_DEVINL void join_part(float& M, float& L, f32x4& o, float m, float l, const f32x4& v) {
    if (l == 0.f) return;                                // nothing there (a NaN sum is not skipped)
    const float mn = fmaxf(M, m), f0 = exp2_hw(M - mn), f1 = exp2_hw(m - mn);
    M = mn;
    L = L * f0 + l * f1;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = o[i] * f0 + v[i] * f1;
}
// 1 / the sum of a row.  A row that sees no key gives zeros; one that sees keys and has no weights, its scores all -infinity, the formula's
// 0 / 0, NaN.
SEEDMI_DEVINL float inverse_sum(float L, bool sees) { return L != 0.f ? 1.f / L : sees ? __uint_as_float(0x7fc00000u) : 0.f; }
SEEDMI_DEVINL void store_row_quad(bf16_t* dst, float L, bool sees, const f32x4& o) {
    const float inv = inverse_sum(L, sees);
    *(uint2*)dst = make_uint2(pack2bf(o[0] * inv, o[1] * inv), pack2bf(o[2] * inv, o[3] * inv));
}
// Parts that another workgroup of the same launch will read, maybe on another XCD with an L2 of its own: device-scope accesses, which go past
// the L2s on both sides.
SEEDMI_DEVINL void store_pair(float* p, float x, float y, bool device) {
    if (device) {
        const unsigned long long w = (unsigned long long)__float_as_uint(y) << 32 | __float_as_uint(x);
        __hip_atomic_store((unsigned long long*)p, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    } else {
        *(float2*)p = make_float2(x, y);
    }
}
SEEDMI_DEVINL void store_quad(float* p, const f32x4& v, bool device) {
    if (device) {
        store_pair(p, v[0], v[1], true);
        store_pair(p + 2, v[2], v[3], true);
    } else {
        *(f32x4*)p = v;
    }
}
SEEDMI_DEVINL float2 load_pair(const float* p) {
    const unsigned long long w = __hip_atomic_load((const unsigned long long*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((unsigned)w), __uint_as_float((unsigned)(w >> 32)));
}
// The last workgroup of a unit to get here joins the unit's rows, in the order of their parts whoever is last: no second launch.  Rows
// first .. + n of the group that starts at token `base`, key head kvh; token t of the group sees seen0 + t * seen_step keys (or none).  Every
// part's stores are past the L2s (waited for) before the workgroup's arrival is counted; the counter wraps to zero with the last arrival.
// Workgroups wait for nobody.
template <int HD>
SEEDMI_DEVINL void join_in_place(const AttnArgs& a, int unit, int base, int kvh, int first, int n, int seen0, int seen_step, float* lds) {
    constexpr int LPR = HD / 4, SLOTS = 256 / LPR, BATCH = 4;
    __shared__ unsigned s_last;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // this wave's stores have reached memory ...
    __syncthreads();                                     // ... and so have the other waves'
    if (threadIdx.x == 0) s_last = atomicInc(a.arrivals + unit, a.unit_blocks - 1) == a.unit_blocks - 1;
    __syncthreads();
    if (!s_last) return;
    asm volatile("" ::: "memory");
    const int c = threadIdx.x % LPR, slot = threadIdx.x / LPR;
    int jw = SLOTS;                                      // threads that share a row's parts: all of them for one row, one each from SLOTS rows on
    while (jw > 1 && jw * n > SLOTS) jw >>= 1;
    const int w = slot % jw, rows_at_once = SLOTS / jw;
    for (int i0 = 0; i0 < n; i0 += rows_at_once) {
        const int r = first + i0 + slot / jw;
        const bool on = r < first + n;
        const int token = base + r / a.GH, head = kvh * a.GH + r % a.GH;
        const long long row = (long long)token * a.H + head;
        float M = LOWEST, L = 0.f;
        f32x4 o = (f32x4){0.f, 0.f, 0.f, 0.f};
        if (on) {
            for (int q = w; q < a.parts; q += BATCH * jw) {
                float2 ml[BATCH], x[BATCH], y[BATCH];
#pragma unroll
                for (int k = 0; k < BATCH; ++k) {
                    const long long at = (long long)min(q + k * jw, a.parts - 1) * a.rows + row;
                    ml[k] = load_pair((const float*)(a.ml_part + at));
                    x[k] = load_pair(a.o_part + at * HD + 4 * c);
                    y[k] = load_pair(a.o_part + at * HD + 4 * c + 2);
                }
#pragma unroll
                for (int k = 0; k < BATCH; ++k)
                    if (q + k * jw < a.parts) join_part(M, L, o, ml[k].x, ml[k].y, (f32x4){x[k].x, x[k].y, y[k].x, y[k].y});
            }
        }
        if (jw > 1) {
            f32x4* so = (f32x4*)lds;                     // [SLOTS][LPR], then (M, L) of each slot
            float2* sl = (float2*)(lds + 1024);
            __syncthreads();
            so[threadIdx.x] = o;
            if (c == 0) sl[slot] = make_float2(M, L);
            __syncthreads();
            if (w == 0)
                for (int k = 1; k < jw; ++k) join_part(M, L, o, sl[slot + k].x, sl[slot + k].y, so[threadIdx.x + k * LPR]);
        }
        if (on && w == 0) store_row_quad(a.out + (size_t)token * a.ldo + head * HD + 4 * c, L, seen0 + r / a.GH * seen_step > 0, o);
    }
}

// ---- few query rows per group (decode, drafted tokens, a shared prefix): bound by the bytes of the cache.
// Bytes: 2 rows of HD values per key and key head, once; 4 HD flops per (row, key) are far below what they cost up to some 100 rows.
// 32 x 32 heads: 4096 rows each 183 us (8-bit, 6.05 TB/s) / 355 us (16-bit, 6.05); slots of different lengths up to 2048
// rows 69 us (5.1); 4 x 8 heads of 23 - 65 thousand rows 82 - 89 us (4.6 - 4.2, with the parts' join); one conversation of 700 rows 8.4 us, latency.
// Workgroup = (group, block of 16 MT rows, key range); its 4 waves take the range's tiles in turn, each with a running softmax of its own,
// and join at the end (eight waves: 4 slots of 65 thousand rows 85 -> 81 us, one short conversation 8.3 -> 9.2).
// S^T = K Q^T (keys are the MFMA's rows: K fragments come straight from memory, one tile ahead in registers), so a
// lane's scores are keys 4 g + r of its query li, which is the layout the P^T operand of O^T = V^T P^T needs: P never leaves registers.
// V is transposed through 8 KiB of LDS that the wave has to itself (no barrier in the loop).
template <int HD, bool MX, int MT>
__global__ __launch_bounds__(256, MT == 2 ? 2 : MX ? 4 : 3) void kv_attention_few_kernel(const AttnArgs a) {
    constexpr int NT = HD / 16, KS = HD / 32;
    constexpr int VBYTES = v_at<HD>(KT, 0);
    __shared__ __attribute__((aligned(16))) char sm[4 * VBYTES];               // >= 4 * 16 * HD floats: the join below
    __shared__ float2 sml[4][16];
    const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // eight items (XCDs) side by side, the row blocks of an item behind each other on its XCD
    unsigned block;
    const AttnPass p = pass_of(a, block);
    const unsigned items = (unsigned)p.groups * p.splits;
    const unsigned blk = block / (8u * p.row_blocks), in = block % (8u * p.row_blocks);
    const unsigned item = blk * 8 + in % 8;
    const int rb = in / 8;
    if (item >= items) return;
    const int G = p.c.G, split = item / p.groups, group = (int)((item % p.groups + (unsigned)split * G) % p.groups);    // (see plan_pass)
    const int slot = group / G, kvh = group % G;
    const int base = p.shared ? 0 : slot * a.T;          // first token row of the group
    const int r0 = rb * 16 * MT, r_end = min(p.group_rows, r0 + 16 * MT);

    const int len = rows_held(p, slot);
    const bool causal = a.causal && !p.shared;
    // rows of keys that a query row sees: all, or up to its own
    const int n_max = causal ? max(0, min(len, len - a.T + (r_end - 1) / a.GH + 1)) : len;
    const int n_min = causal ? max(0, min(len, len - a.T + r0 / a.GH + 1)) : len;
    const int tiles = (n_max + KT - 1) / KT;
    const int per = max((tiles + p.splits - 1) / p.splits, p.per_split);
    const int t_begin = split * per, t_end = min(tiles, t_begin + per);

    const long long row0 = (p.shared ? 0ll : (long long)slot * p.c.slot_rows) + (long long)kvh * p.c.head_rows;
    const RowBuffers rows = row_buffers<HD, MX>(p.c, row0, n_max);
    Tile<HD, MX> t;                                      // (the first tile is on its way while the queries are fetched)
    if (t_begin + wave < t_end) {
        load_v(t, rows, (t_begin + wave) * KT, lane);
        load_k(t, rows, (t_begin + wave) * KT, lane);
    }

    bf16x8 qf[MT][KS];
    int seen[MT];
    float m[MT], ref[MT], l[MT];                         // largest score, reference(), sum
    f32x4 o[MT][NT];
#pragma unroll
    for (int u = 0; u < MT; ++u) {
        const int r = r0 + 16 * u + li;
        const bool on = r < r_end;
        seen[u] = on ? (causal ? len - a.T + r / a.GH + 1 : len) : 0;
        const bf16_t* qp = a.q + (size_t)(base + (on ? r / a.GH : 0)) * a.ldq + (kvh * a.GH + (on ? r % a.GH : 0)) * HD;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int d = MX ? 64 * (ks >> 1) + 16 * g4 + 8 * (ks & 1) : 32 * ks + 8 * g4;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (on) v = *(const uint4*)(qp + d);
            qf[u][ks] = __builtin_bit_cast(bf16x8, v);
        }
        m[u] = -INFINITY;
        ref[u] = l[u] = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n) o[u][n] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    char* lds = sm + wave * VBYTES;
    bool far = false;                                    // (wave-uniform) a reference beyond FAR

    arrived(qf);
#pragma unroll 1
    for (int tile = t_begin + wave; tile < t_end; tile += 4) {
        const int key0 = tile * KT, next0 = (tile + 4 < t_end ? tile + 4 : tiles) * KT;    // (behind the last row: nothing is fetched)
        const bool partial = key0 + KT > n_min;          // (wave-uniform) some row of the block does not see all of the tile
        bool mixed = false;
        lds_fence();
        if (!partial) stage_v<HD, MX, false>(t, lds, lane);
        else mixed = __any(stage_v<HD, MX, true>(t, lds, lane));
        lds_fence();
        load_v(t, rows, next0, lane);                    // the wave's next tile
        f32x4 s[MT][2];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            bf16x8 kf[KS];
#pragma unroll
            for (int j = 0; j < Tile<HD, MX>::KL; ++j) {
                const uint4 w = t.k[kt][j];
                if (MX) {
                    const float sc = mx_scale_f((t.ks[kt] >> (16 * j + 8 * (g4 >> 1))) & 255u);
                    kf[2 * j] = __builtin_bit_cast(bf16x8, make_uint4(mx_unpack2<false>(w.x, sc), mx_unpack2<true>(w.x, sc), mx_unpack2<false>(w.y, sc), mx_unpack2<true>(w.y, sc)));
                    kf[2 * j + 1] = __builtin_bit_cast(bf16x8, make_uint4(mx_unpack2<false>(w.z, sc), mx_unpack2<true>(w.z, sc), mx_unpack2<false>(w.w, sc), mx_unpack2<true>(w.w, sc)));
                } else {
                    kf[j] = __builtin_bit_cast(bf16x8, w);
                }
            }
#pragma unroll
            for (int u = 0; u < MT; ++u) {
                s[u][kt] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) s[u][kt] = seedmi_mfma_16x16x32(kf[ks], qf[u][ks], s[u][kt]);
            }
        }
        load_k(t, rows, next0, lane);
        bf16x8 pf[MT];
#pragma unroll
        for (int u = 0; u < MT; ++u) {
            if (partial) {
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (key0 + 16 * kt + 4 * g4 + r >= seen[u]) s[u][kt][r] = -INFINITY;
            }
            float tm = max3(max3(s[u][0][0], s[u][0][1], s[u][0][2]), max3(s[u][0][3], s[u][1][0], s[u][1][1]), max2(s[u][1][2], s[u][1][3]));
            tm = rows_max(tm) * a.c2;
            if (__any(tm > m[u])) {                      // a new maximum (a NaN is none): what is summed so far is scaled down
                const float mn = fmaxf(m[u], tm), rn = reference(mn);
                const float f = m[u] == -INFINITY ? 0.f : exp2_hw(ref[u] - rn);
                l[u] *= f;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[u][n][r] *= f;
                m[u] = mn;
                ref[u] = rn;
                far |= __any(fabsf(rn) >= FAR);
            }
            if (far) {
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[u][kt][r] = rounded(s[u][kt][r] * a.c2);
            }
            const float mul = far ? 1.f : a.c2;
            float e[2][4];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int r = 0; r < 4; ++r) e[kt][r] = exp2_hw(fmaf(s[u][kt][r], mul, -ref[u]));
            const uint4 w = make_uint4(pack2bf(e[0][0], e[0][1]), pack2bf(e[0][2], e[0][3]), pack2bf(e[1][0], e[1][1]), pack2bf(e[1][2], e[1][3]));
            l[u] = add_probabilities(w, l[u]);
            pf[u] = __builtin_bit_cast(bf16x8, w);
        }
        if (mixed) {
            // Values that are not finite in a tile that some rows do not see whole: 0 * inf must not reach a row that does not see the key.
            // They are added here to the rows that do, and taken out of the image.
            lds_fence();
            const int ln = fresh_lane(), g = ln >> 4;    // (cold: no address of this block is kept across the loop)
#pragma unroll 1
            for (int j = 0; j < KT; ++j) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint2 w = *(const uint2*)(lds + v_at<HD>(j, 2 * n) + 8 * g);
                    const uint32_t h[4] = {w.x & 0xffffu, w.x >> 16, w.y & 0xffffu, w.y >> 16};
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int u = 0; u < MT; ++u)
                            if (bad16(h[r]) && key0 + j < seen[u]) o[u][n][r] += bf2f((bf16_t)h[r]);
                }
            }
            lds_fence();
#pragma unroll 1
            for (int i = 16 * ln; i < VBYTES; i += 1024) {
                uint32_t* w = (uint32_t*)(lds + i);
#pragma unroll
                for (int d = 0; d < 4; ++d) w[d] = clean_word(w[d]);
            }
            lds_fence();
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const bf16x8 vf = v_frag<HD>(lds, n, lane);
#pragma unroll
            for (int u = 0; u < MT; ++u) o[u][n] = seedmi_mfma_16x16x32(vf, pf[u], o[u][n]);
        }
    }

    // the four waves' (m, l, o) joined, one block of 16 rows at a time; thread = (row, HD / 16 channels)
    float* so = (float*)sm;
#pragma unroll
    for (int u = 0; u < MT; ++u) {
        const float lsum = rows_sum(l[u]), mr = m[u] == -INFINITY ? LOWEST : ref[u];
        __syncthreads();
        if (g4 == 0) sml[wave][li] = make_float2(mr, lsum);
        __syncthreads();
        float M = LOWEST;                                // (finite: a sum that is NaN stays NaN, one that is 0 is left out)
#pragma unroll
        for (int w = 0; w < 4; ++w) M = fmaxf(M, sml[w][li].x);
        const float f = exp2_hw(mr - M);
        // channel quads 4 (4 n + g) of row li, XOR-ed with the row
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            f32x4 v;
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = lsum == 0.f ? 0.f : o[u][n][r] * f;
            *(f32x4*)(so + (wave * 16 + li) * HD + (((4 * n + g4) ^ li) << 2)) = v;
        }
        __syncthreads();
        const int row = tid >> 4, part = tid & 15;
        const int r = r0 + 16 * u + row;
        float L = 0.f, Mr = LOWEST;
#pragma unroll
        for (int w = 0; w < 4; ++w) Mr = fmaxf(Mr, sml[w][row].x);
#pragma unroll
        for (int w = 0; w < 4; ++w) L += sml[w][row].y * exp2_hw(sml[w][row].x - Mr);
        if (r < r_end) {
            constexpr int Q = HD / 64;                   // quads of a thread
            const int token = base + r / a.GH, head = kvh * a.GH + r % a.GH;
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                const int quad = part * Q + i;
                f32x4 v = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const f32x4 x = *(const f32x4*)(so + (w * 16 + row) * HD + ((quad ^ row) << 2));
#pragma unroll
                    for (int d = 0; d < 4; ++d) v[d] += x[d];
                }
                if (a.parts == 1) {
                    const float inv = inverse_sum(L, (causal ? len - a.T + r / a.GH + 1 : len) > 0);
                    *(uint2*)(a.out + (size_t)token * a.ldo + head * HD + 4 * quad) = make_uint2(pack2bf(v[0] * inv, v[1] * inv), pack2bf(v[2] * inv, v[3] * inv));
                } else {
                    const long long at = (long long)(p.part0 + split) * a.rows + (long long)token * a.H + head;
                    if (L != 0.f) store_quad(a.o_part + at * HD + 4 * quad, v, a.arrivals != nullptr);
                    if (part == 0 && i == 0) store_pair((float*)(a.ml_part + at), Mr, L, a.arrivals != nullptr);
                }
            }
        }
    }
    if (a.arrivals) {
        const int unit = a.unit_rows ? kvh : group * p.row_blocks + rb;
        const int first = a.unit_rows ? 0 : r0, n_rows = a.unit_rows ? a.unit_rows : r_end - r0;
        // (a unit of two passes: every row sees the prefix)
        join_in_place<HD>(a, unit, a.unit_rows ? 0 : base, kvh, first, n_rows, a.unit_rows ? 1 : causal ? len - a.T + 1 : len,
                          a.unit_rows ? 0 : causal, (float*)sm);
    }
}

// ---- many query rows per group (prompt chunks, a prefix that many slots share): bound by the matrix and vector pipes.
// Workgroup = (group, block of 64 MT rows, key range), wave = 16 MT rows; 64-key tiles of K and V are widened to 16 bits once and shared
// through a double-buffered LDS image, one barrier per tile; the next tile's bytes are in registers meanwhile, so that neither the load nor
// the widening sits between two tiles.  8 x 40 heads, 100 new rows behind 549: 40 us (8-bit) / 37 us (16-bit).
constexpr int KT2 = 64;

template <int HD, bool MX>
struct Stage {                                           // a thread's part of a 64-key tile of K and of V: HD * 4 / RB rows ... 16 bytes each
    static constexpr int RB = MX ? HD : 2 * HD;
    static constexpr int LPR = RB / 16;                  // threads of a row
    static constexpr int L = KT2 * LPR / 256;            // 16-byte loads per thread and operand
    uint4 k[L], v[L];
    uint32_t ks[L], vs[L];
};
template <int HD, bool MX>
SEEDMI_DEVINL void stage_load(Stage<HD, MX>& t, const RowBuffers& b, int key0, int tid) {
    using S = Stage<HD, MX>;
    const int row = tid / S::LPR, c = tid % S::LPR;
#pragma unroll
    for (int j = 0; j < S::L; ++j) {
        const int r = row + j * (256 / S::LPR);
        t.k[j] = load16(b.k, r * S::RB + 16 * c, key0 * S::RB);
        t.v[j] = load16(b.v, r * S::RB + 16 * c, key0 * S::RB);
        if (MX) {
            t.ks[j] = load_scale<HD>(b.ks, r, c / 2, key0 * (HD / 32));
            t.vs[j] = load_scale<HD>(b.vs, r, c / 2, key0 * (HD / 32));
        }
    }
}
template <int HD, bool MX>
SEEDMI_DEVINL void stage_store(const Stage<HD, MX>& t, char* kl, char* vl, int tid) {
    using S = Stage<HD, MX>;
    auto put = [](char* dst, uint4 w, uint32_t sb, int blk) {
        if (MX) {
            const float s = scale_of<HD>(sb, blk);
            *(uint4*)dst = make_uint4(mx_unpack2<false>(w.x, s), mx_unpack2<true>(w.x, s), mx_unpack2<false>(w.y, s), mx_unpack2<true>(w.y, s));
            *(uint4*)(dst + 16) = make_uint4(mx_unpack2<false>(w.z, s), mx_unpack2<true>(w.z, s), mx_unpack2<false>(w.w, s), mx_unpack2<true>(w.w, s));
        } else {
            *(uint4*)dst = make_uint4(w.x, w.y, w.z, w.w);
        }
    };
#pragma unroll
    for (int j = 0; j < S::L; ++j) {
        const int row = j * (256 / S::LPR) + tid / S::LPR, c = tid % S::LPR;
        put(kl + k_at<HD>(row, MX ? 2 * c : c), t.k[j], MX ? t.ks[j] : 0u, c / 2);
        put(vl + v_at<HD>(row, MX ? 2 * c : c), t.v[j], MX ? t.vs[j] : 0u, c / 2);
    }
}

template <int HD, bool MX, int MT>
__global__ __launch_bounds__(256, 2) void kv_attention_many_kernel(const AttnArgs a) {
    constexpr int NT = HD / 16, KS = HD / 32;
    constexpr int KB = k_at<HD>(KT2, 0), VB = v_at<HD>(KT2, 0);          // bytes of the images
    __shared__ __attribute__((aligned(16))) char sm[2 * KB + 2 * VB];    // K0 K1 V0 V1
    const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    unsigned block;
    const AttnPass p = pass_of(a, block);
    const unsigned items = (unsigned)p.groups * p.splits;
    const unsigned blk = block / (8u * p.row_blocks), in = block % (8u * p.row_blocks);
    const unsigned item = blk * 8 + in % 8;
    const int rb = p.row_blocks - 1 - (int)(in / 8);     // (causal: the longest ranges first)
    if (item >= items) return;
    const int G = p.c.G, split = item / p.groups, group = (int)((item % p.groups + (unsigned)split * G) % p.groups);    // (see plan_pass)
    const int slot = group / G, kvh = group % G;
    const int base = p.shared ? 0 : slot * a.T;
    const int r0 = rb * 64 * MT, r_end = min(p.group_rows, r0 + 64 * MT);

    const int len = rows_held(p, slot);
    const bool causal = a.causal && !p.shared;
    const int n_max = causal ? max(0, min(len, len - a.T + (r_end - 1) / a.GH + 1)) : len;
    const int tiles = (n_max + KT2 - 1) / KT2;
    const int per = max((tiles + p.splits - 1) / p.splits, p.per_split);
    const int t_begin = split * per, t_end = min(tiles, t_begin + per);
    // what the rows of this wave see at least and at most (its rows may lie beyond the group's end)
    const int w0 = r0 + 16 * MT * wave, w1 = min(r_end - 1, w0 + 16 * MT - 1);
    const int wave_max = w0 >= r_end ? 0 : causal ? len - a.T + w1 / a.GH + 1 : len;
    const int wave_min = w0 >= r_end ? 0 : causal ? len - a.T + w0 / a.GH + 1 : len;

    const long long row0 = (p.shared ? 0ll : (long long)slot * p.c.slot_rows) + (long long)kvh * p.c.head_rows;
    using S = Stage<HD, MX>;
    const RowBuffers rows = row_buffers<HD, MX>(p.c, row0, n_max);
    S st;                                                // (the first tile is on its way while the queries are fetched)
    if (t_begin < t_end) stage_load(st, rows, t_begin * KT2, tid);

    bf16x8 qf[MT][KS];
    int seen[MT];
    float m[MT], ref[MT], l[MT];                         // largest score, reference(), sum
    f32x4 o[MT][NT];
#pragma unroll
    for (int u = 0; u < MT; ++u) {
        const int r = w0 + 16 * u + li;
        const bool on = r < r_end;
        seen[u] = on ? (causal ? len - a.T + r / a.GH + 1 : len) : 0;
        const bf16_t* qp = a.q + (size_t)(base + (on ? r / a.GH : 0)) * a.ldq + (kvh * a.GH + (on ? r % a.GH : 0)) * HD;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (on) v = *(const uint4*)(qp + 32 * ks + 8 * g4);
            qf[u][ks] = __builtin_bit_cast(bf16x8, v);
        }
        m[u] = -INFINITY;
        ref[u] = l[u] = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n) o[u][n] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    bool far = false;                                    // (wave-uniform) a reference beyond FAR
    arrived(qf);
    if (t_begin < t_end) {
        stage_store(st, sm, sm + 2 * KB, tid);
        stage_load(st, rows, (t_begin + 1 < t_end ? t_begin + 1 : tiles) * KT2, tid);
    }
    __syncthreads();
#pragma unroll 1
    for (int tile = t_begin; tile < t_end; ++tile) {
        const int key0 = tile * KT2, cur = (tile - t_begin) & 1;
        char* kl = sm + cur * KB;
        char* vl = sm + 2 * KB + cur * VB;
        bool mixed = false;
        if (key0 + KT2 > n_max || (causal && key0 + KT2 > len - a.T + r0 / a.GH + 1)) {          // (uniform) some row does not see it all
            bool bad = false;
#pragma unroll 1
            for (int i = 16 * tid; i < KT2 * 2 * HD; i += 4096) bad |= bad_words(*(const uint4*)(vl + v_at<HD>(i / (2 * HD), i % (2 * HD) / 16)));
            mixed = __syncthreads_or(bad) != 0;
        }
        f32x4 s[MT][4];
        const bool live = key0 < wave_max;               // (wave-uniform)
        if (live) {
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                bf16x8 kf[KS];
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) kf[ks] = *(const bf16x8*)(kl + k_at<HD>(16 * kt + li, 4 * ks + g4));
#pragma unroll
                for (int u = 0; u < MT; ++u) {
                    s[u][kt] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) s[u][kt] = seedmi_mfma_16x16x32(kf[ks], qf[u][ks], s[u][kt]);
                }
            }
        }
        // the next tile into the other buffer (read last before the barrier that ended the previous tile), the one after it requested
        if (tile + 1 < t_end) {
            stage_store(st, sm + (cur ^ 1) * KB, sm + 2 * KB + (cur ^ 1) * VB, tid);
            stage_load(st, rows, (tile + 2 < t_end ? tile + 2 : tiles) * KT2, tid);
        }
        bf16x8 pf[MT][2];
        if (live) {
#pragma unroll
            for (int u = 0; u < MT; ++u) {
                if (key0 + KT2 > wave_min) {
#pragma unroll
                    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (key0 + 16 * kt + 4 * g4 + r >= seen[u]) s[u][kt][r] = -INFINITY;
                }
                float tm = -INFINITY;
#pragma unroll
                for (int kt = 0; kt < 4; ++kt) tm = max3(max3(tm, s[u][kt][0], s[u][kt][1]), s[u][kt][2], s[u][kt][3]);
                tm = rows_max(tm) * a.c2;
                if (__any(tm > m[u])) {
                    const float mn = fmaxf(m[u], tm), rn = reference(mn);
                    const float f = m[u] == -INFINITY ? 0.f : exp2_hw(ref[u] - rn);
                    l[u] *= f;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[u][n][r] *= f;
                    m[u] = mn;
                    ref[u] = rn;
                    far |= __any(fabsf(rn) >= FAR);
                }
                if (far) {
#pragma unroll
                    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[u][kt][r] = rounded(s[u][kt][r] * a.c2);
                }
                const float mul = far ? 1.f : a.c2;
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                    float e[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) e[j] = exp2_hw(fmaf(s[u][2 * kk + (j >> 2)][j & 3], mul, -ref[u]));
                    const uint4 w = make_uint4(pack2bf(e[0], e[1]), pack2bf(e[2], e[3]), pack2bf(e[4], e[5]), pack2bf(e[6], e[7]));
                    l[u] = add_probabilities(w, l[u]);
                    pf[u][kk] = __builtin_bit_cast(bf16x8, w);
                }
            }
        }
        if (mixed) {                                     // see kv_attention_few_kernel
            if (live) {
                const int g = fresh_lane() >> 4;
#pragma unroll 1
                for (int j = 0; j < KT2; ++j) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const uint2 w = *(const uint2*)(vl + v_at<HD>(j, 2 * n) + 8 * g);
                        const uint32_t h[4] = {w.x & 0xffffu, w.x >> 16, w.y & 0xffffu, w.y >> 16};
#pragma unroll
                        for (int r = 0; r < 4; ++r)
#pragma unroll
                            for (int u = 0; u < MT; ++u)
                                if (bad16(h[r]) && key0 + j < seen[u]) o[u][n][r] += bf2f((bf16_t)h[r]);
                    }
                }
            }
            __syncthreads();
#pragma unroll 1
            for (int i = 4 * tid; i < VB; i += 1024) *(uint32_t*)(vl + i) = clean_word(*(uint32_t*)(vl + i));
            __syncthreads();
        }
        if (live) {
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const bf16x8 vf = v_frag<HD>(vl + v_at<HD>(32 * kk, 0), n, lane);
#pragma unroll
                    for (int u = 0; u < MT; ++u) o[u][n] = seedmi_mfma_16x16x32(vf, pf[u][kk], o[u][n]);
                }
        }
        __syncthreads();
    }

#pragma unroll
    for (int u = 0; u < MT; ++u) {
        const float L = rows_sum(l[u]);
        const int r = w0 + 16 * u + li;
        if (r >= r_end) continue;
        const int token = base + r / a.GH, head = kvh * a.GH + r % a.GH;
        if (a.parts == 1) {
            const float inv = inverse_sum(L, seen[u] > 0);
            bf16_t* op = a.out + (size_t)token * a.ldo + head * HD + 4 * g4;
#pragma unroll
            for (int n = 0; n < NT; ++n)
                *(uint2*)(op + 16 * n) = make_uint2(pack2bf(o[u][n][0] * inv, o[u][n][1] * inv), pack2bf(o[u][n][2] * inv, o[u][n][3] * inv));
        } else {
            const long long at = (long long)(p.part0 + split) * a.rows + (long long)token * a.H + head;
            if (L != 0.f) {
#pragma unroll
                for (int n = 0; n < NT; ++n) *(f32x4*)(a.o_part + at * HD + 16 * n + 4 * g4) = o[u][n];
            }
            if (g4 == 0) a.ml_part[at] = make_float2(m[u] == -INFINITY ? LOWEST : ref[u], L);
        }
    }
}

// ---- hundreds of query rows per group: bound by what two waves per SIMD can issue (matrix products, exponentials, and every other
// instruction of the softmax and of widening a tile).
// Workgroup = (group, block of 256 rows, key range), two halves of four waves; wave = 32 rows on 32 x 32 x 16 products (half the instructions
// of 16 x 16 ones, and a lane has one query: S^T = K Q^T puts keys 8 (r >> 2) + 4 h + (r & 3) of query lane & 31 into register r, h = lane >> 5,
// which eight at a time are the P^T operand of O^T = V^T P^T).  A tile costs a wave a MATRIX phase (the product with the previous tile's
// values, then the scores of this one) and a VECTOR phase (softmax, staging) of about the same length.  The halves run one phase apart, so
// that on every SIMD one wave is in its matrix phase while the other is in its vector phase; a barrier ends each phase.  Phase 2 t: half 0
// multiplies (values of t - 1, keys of t); phase 2 t + 1: half 1 does.  Keys of tile t are read in phases 2 t and 2 t + 1, values in 2 t + 2
// and 2 t + 3; each half stages its 32 rows of a tile in its vector phases: half h, after the scores of tile t, keys of t + 1 + h and
// values of t + h - two LDS buffers each, always written after their last reader's barrier.
// Tiles that every row of the block sees whole take a loop without masks and case distinctions (a lone wave issues an instruction every
// five to six cycles, scalar ones too: it is their number that counts).
// 2 x 32 heads, 2048 new rows each in caches of up to 4001: 138 GF in 192 - 196 us, 717 - 703 TFLOP/s (both slots at 4001 rows: 246 us, 811); a
// plain 8192^3 product of the type reaches 1284 and more.  With one phase's work taken out (kernel at 195 us): matrix phases alone 135 us, vector phases
// alone 162; without the requests for the next tiles 160.
// On 16 x 16 x 32 products and one loop for all tiles the same kernel took 232 us, unphased with two workgroups per CU 244.
typedef __attribute__((ext_vector_type(16))) float f32x16;
SEEDMI_DEVINL f32x16 mfma_32x32x16(bf16x8 a, bf16x8 b, f32x16 c) {
#ifdef SEEDMI_F16
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(hw_f16x8, a), __builtin_bit_cast(hw_f16x8, b), c, 0, 0, 0);
#else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
#endif
}
template <int HD>
SEEDMI_DEVINL constexpr int w_at(int row, int c) { return row * (2 * HD + 64) + 16 * c; }      // value rows here: 64 bytes of 4 rows at a time

template <int HD, bool MX>
struct HalfStage {                                       // a thread's part of 32 rows of K and V
    static constexpr int RB = MX ? HD : 2 * HD;
    static constexpr int LPR = RB / 16;
    static constexpr int L = (32 * LPR + 255) / 256;     // 16-byte loads per thread (8-bit rows of 64: by half of the threads)
    uint4 k[L], v[L];
    uint32_t ks[L], vs[L];
};
struct WholeTile { static constexpr bool value = true; };                // every row of the block sees all of the tile
struct AnyTile { static constexpr bool value = false; };

template <int HD, bool MX>
__global__ __launch_bounds__(512) void kv_attention_phased_kernel(const AttnArgs a) {
    constexpr int NT = HD / 32, KS = HD / 16;
    constexpr int KB = k_at<HD>(KT2, 0), VB = w_at<HD>(KT2, 0);          // bytes of the images
    __shared__ __attribute__((aligned(16))) char sm[2 * KB + 4 * VB];    // K0 K1, V0 V1, raw V0 V1
    __shared__ int s_bad;                                // a tile that some row does not see whole held a value that is not finite
    const int tid = threadIdx.x, lane = tid & 63, lq = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = wave >> 2, ht = tid & 255;
    unsigned block;
    const AttnPass p = pass_of(a, block);
    const unsigned items = (unsigned)p.groups * p.splits;
    const unsigned blk = block / (8u * p.row_blocks), in = block % (8u * p.row_blocks);
    const unsigned item = blk * 8 + in % 8;
    const int rb = p.row_blocks - 1 - (int)(in / 8);     // (causal: the longest ranges first)
    if (item >= items) return;
    const int G = p.c.G, split = item / p.groups, group = (int)((item % p.groups + (unsigned)split * G) % p.groups);    // (see plan_pass)
    const int slot = group / G, kvh = group % G;
    const int base = p.shared ? 0 : slot * a.T;
    const int r0 = rb * 256, r_end = min(p.group_rows, r0 + 256);

    const int len = rows_held(p, slot);
    const bool causal = a.causal && !p.shared;
    const int n_max = causal ? max(0, min(len, len - a.T + (r_end - 1) / a.GH + 1)) : len;
    const int n_min = causal ? len - a.T + r0 / a.GH + 1 : len;
    const int tiles = (n_max + KT2 - 1) / KT2;
    const int per = max((tiles + p.splits - 1) / p.splits, p.per_split);
    const int t0 = split * per, n = max(0, min(tiles, t0 + per) - t0);   // first tile, number of tiles
    const int w0 = r0 + 32 * wave, w1 = min(r_end - 1, w0 + 31);
    const bool active = w0 < r_end;                      // the wave has rows
    const int wave_max = !active ? 0 : causal ? len - a.T + w1 / a.GH + 1 : len;
    const int wave_min = !active ? 0 : causal ? len - a.T + w0 / a.GH + 1 : len;

    const int r = w0 + lq;                               // this lane's query row
    const bool on = r < r_end;
    const int token = base + (on ? r / a.GH : 0), head = kvh * a.GH + (on ? r % a.GH : 0);
    const int seen = on ? (causal ? len - a.T + r / a.GH + 1 : len) : 0;
    const long long row0 = (p.shared ? 0ll : (long long)slot * p.c.slot_rows) + (long long)kvh * p.c.head_rows;
    using S = HalfStage<HD, MX>;
    const RowBuffers rows = row_buffers<HD, MX>(p.c, row0, n_max);
    const int srow = 32 * half + ht / S::LPR, schunk = ht % S::LPR;      // the thread's first row of a tile and its 16-byte piece of it
    const bool stages = 32 * S::LPR >= 256 || ht < 32 * S::LPR;

    constexpr int KP = k_at<HD>(1, 0), VP = w_at<HD>(1, 0);              // row pitches of the images
    S st;                                                // (a second set, requested two tiles ahead: no faster)
    // tiles from n on: behind the last row, nothing is fetched
    auto load_rows = [&](uint4 (&w)[S::L], uint32_t (&sc)[S::L], const __amdgpu_buffer_rsrc_t& b, const __amdgpu_buffer_rsrc_t& sb, int t) __attribute__((always_inline)) {
        if (!stages) return;
        const int key0 = (t < n ? t0 + t : tiles) * KT2;
#pragma unroll
        for (int j = 0; j < S::L; ++j) {
            const int row = srow + j * (256 / S::LPR);
            w[j] = load16(b, row * S::RB + 16 * schunk, key0 * S::RB);
            if (MX) sc[j] = load_scale<HD>(sb, row, schunk / 2, key0 * (HD / 32));
        }
    };
    // raw: where a value tile that some row does not see whole leaves its rows as they are; the image then holds zeros in place of what is not
    // finite (0 * inf must not reach a row that does not see the key; the rows that do take it from the raw rows)
    auto store_rows = [&](const uint4 (&w)[S::L], const uint32_t (&sc)[S::L], char* dst, int pitch, char* raw) __attribute__((always_inline)) {
        if (!stages) return;
        bool bad = false;
        auto put = [&](int at, uint4 x) {
            if (raw) {
                *(uint4*)(raw + at) = x;
                bad |= bad_words(x);
                x = make_uint4(clean_word(x.x), clean_word(x.y), clean_word(x.z), clean_word(x.w));
            }
            *(uint4*)(dst + at) = x;
        };
#pragma unroll
        for (int j = 0; j < S::L; ++j) {
            const int at = (srow + j * (256 / S::LPR)) * pitch + (MX ? 32 : 16) * schunk;
            if (MX) {
                const float s = scale_of<HD>(sc[j], schunk / 2);
                put(at, make_uint4(mx_unpack2<false>(w[j].x, s), mx_unpack2<true>(w[j].x, s), mx_unpack2<false>(w[j].y, s), mx_unpack2<true>(w[j].y, s)));
                put(at + 16, make_uint4(mx_unpack2<false>(w[j].z, s), mx_unpack2<true>(w[j].z, s), mx_unpack2<false>(w[j].w, s), mx_unpack2<true>(w[j].w, s)));
            } else {
                put(at, make_uint4(w[j].x, w[j].y, w[j].z, w[j].w));
            }
        }
        if (raw && bad) s_bad = 1;
    };
    auto kbuf = [&](int t) { return sm + (t & 1) * KB; };
    auto vbuf = [&](int t) { return sm + 2 * KB + (t & 1) * VB; };
    auto partial_tile = [&](int t) { return (t0 + t + 1) * KT2 > n_min; };               // some row of the block does not see all of it
    auto vraw = [&](int t) { return partial_tile(t) ? sm + 2 * KB + (2 + (t & 1)) * VB : nullptr; };

    // the tiles staged ahead of the first phase (half 1 is one vector phase ahead) and the queries are requested together
    S first;
    if (tid == 0) s_bad = 0;
    if (n > 0) {
        load_rows(first.k, first.ks, rows.k, rows.ks, 0);
        if (half) {
            load_rows(st.k, st.ks, rows.k, rows.ks, 1);
            load_rows(first.v, first.vs, rows.v, rows.vs, 0);
        }
    }
    bf16x8 qf[1][KS];
    {
        const bf16_t* qp = a.q + (size_t)token * a.ldq + head * HD + 8 * h;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (on) v = *(const uint4*)(qp + 16 * ks);
            qf[0][ks] = __builtin_bit_cast(bf16x8, v);
        }
    }
    float m = -INFINITY, nref = 0.f, l = 0.f;            // largest score, -reference() (as the exponents take it), sum
    unsigned long long far = 0;                          // rows with a reference beyond FAR: their wave always takes the branch of a new
    float mul = a.c2;                                    // maximum, the others have no second one (it costs 4 us of 192)
    f32x16 o[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int d = 0; d < 16; ++d) o[i][d] = 0.f;
    arrived(qf);
    __syncthreads();                                     // (s_bad is set)
    if (n > 0) {
        store_rows(first.k, first.ks, kbuf(0), KP, nullptr);
        if (half) {
            store_rows(st.k, st.ks, kbuf(1), KP, nullptr);
            store_rows(first.v, first.vs, vbuf(0), VP, vraw(0));
        }
        load_rows(st.k, st.ks, rows.k, rows.ks, 1 + half);
        load_rows(st.v, st.vs, rows.v, rows.vs, half);
    }
    __syncthreads();

    bf16x8 pf[4];                                        // P^T of a tile, 16 keys each
    const int vlane = w_at<HD>(4 * h + ((lane & 15) >> 2), 0) + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
    auto values = [&](int t) __attribute__((always_inline)) {                           // o += P V for the tile whose probabilities are in pf
        const char* vl = vbuf(t) + vlane;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                // channels 32 i + (lane & 31), keys 16 ks + 4 h + (j & 3) + 8 (j >> 2)
                const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vl + w_at<HD>(16 * ks, 4 * i)));
                const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vl + w_at<HD>(16 * ks + 8, 4 * i)));
                const uint2 lo = __builtin_bit_cast(uint2, x), hi = __builtin_bit_cast(uint2, y);
                o[i] = mfma_32x32x16(__builtin_bit_cast(bf16x8, make_uint4(lo.x, lo.y, hi.x, hi.y)), pf[ks], o[i]);
            }
    };
    auto values_not_finite = [&](int t) __attribute__((always_inline)) {                // see kv_attention_few_kernel
        if (__builtin_amdgcn_readfirstlane(s_bad) == 0) return;
        const int hh = fresh_lane() >> 5;
        const char* rl = sm + 2 * KB + (2 + (t & 1)) * VB;
#pragma unroll 1
        for (int j = 0; j < KT2; ++j) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint2 w = *(const uint2*)(rl + w_at<HD>(j, 4 * i + e) + 8 * hh);
                    const uint32_t x[4] = {w.x & 0xffffu, w.x >> 16, w.y & 0xffffu, w.y >> 16};
#pragma unroll
                    for (int d = 0; d < 4; ++d)
                        if (bad16(x[d]) && (t0 + t) * KT2 + j < seen) o[i][4 * e + d] += bf2f((bf16_t)x[d]);
                }
        }
    };
    const int klane = k_at<HD>(lq, h);
    f32x16 s[2];
    auto scores = [&](int t) __attribute__((always_inline)) {
        const char* kl = kbuf(t) + klane;
#pragma unroll
        for (int d = 0; d < 16; ++d) s[0][d] = s[1][d] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) s[kt] = mfma_32x32x16(*(const bf16x8*)(kl + k_at<HD>(32 * kt, 2 * ks)), qf[0][ks], s[kt]);
    };
    auto softmax = [&](int key0, bool masked) __attribute__((always_inline)) {
        if (masked) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int d = 0; d < 16; ++d)
                    if (key0 + 32 * kt + 8 * (d >> 2) + 4 * h + (d & 3) >= seen) s[kt][d] = -INFINITY;
        }
        float tm = max2(s[0][0], s[1][0]);
#pragma unroll
        for (int d = 1; d < 16; ++d) tm = max3(tm, s[0][d], s[1][d]);
        auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(tm), __float_as_uint(tm), false, false);
        tm = max2(__uint_as_float(w[0]), __uint_as_float(w[1])) * a.c2;
        if ((__ballot(tm > m) | far) != 0) {             // (a NaN among the scores is in the sums, whatever the maximum)
            const float mn = fmaxf(m, tm), rn = reference(mn);
            const float f = m == -INFINITY ? 0.f : exp2_hw(-nref - rn);
            l *= f;
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int d = 0; d < 16; ++d) o[i][d] *= f;
            m = mn;
            nref = -rn;
            far |= __ballot(fabsf(rn) >= FAR);
            if (far) {
                mul = 1.f;
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int d = 0; d < 16; ++d) s[kt][d] = rounded(s[kt][d] * a.c2);
            }
        }
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            float e[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = exp2_hw(fmaf(s[ks >> 1][8 * (ks & 1) + j], mul, nref));
            const uint4 w = make_uint4(pack2bf(e[0], e[1]), pack2bf(e[2], e[3]), pack2bf(e[4], e[5]), pack2bf(e[6], e[7]));
            l = add_probabilities(w, l);
            pf[ks] = __builtin_bit_cast(bf16x8, w);
        }
    };
    auto step = [&](auto whole, int t) __attribute__((always_inline)) {                 // matrix phase and vector phase of tile t
        constexpr bool W = decltype(whole)::value;       // (tiles before a whole one are whole)
        const int key0 = (t0 + t) * KT2;
        const bool live = W ? active : key0 < wave_max;  // (wave-uniform; tiles are in order: once dead, dead to the end)
        __builtin_amdgcn_s_setprio(1);
        if (W) {
            if (live) {
                values(t - 1);
                scores(t);
                // fragments are read four products ahead of their use (left alone, the compiler reads two, waits, and multiplies twice)
                __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
                for (int i = 0; i < 4 * NT - 4; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                }
#pragma unroll
                for (int i = 0; i < 2 * KS; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
            }
        } else {
            if (t > 0 && key0 - KT2 < wave_max) {
                values(t - 1);
                if (partial_tile(t - 1)) values_not_finite(t - 1);
            }
            if (live) scores(t);
        }
        __builtin_amdgcn_s_setprio(0);
        __syncthreads();
        store_rows(st.k, st.ks, kbuf(t + 1 + half), KP, nullptr);
        store_rows(st.v, st.vs, vbuf(t + half), VP, W ? nullptr : vraw(t + half));
        load_rows(st.k, st.ks, rows.k, rows.ks, t + 2 + half);
        load_rows(st.v, st.vs, rows.v, rows.vs, t + 1 + half);
        if (live) softmax(key0, W ? false : key0 + KT2 > wave_min);
        __syncthreads();
    };
    // the whole tiles, less the last of them: a vector phase stages values of up to one tile later
    const int whole = min(n, n_min / KT2 - t0) - 1;
    if (half) __syncthreads();                           // phase 0 belongs to half 0
#pragma unroll 1
    for (int t = 0; t < n;) {
        step(AnyTile(), t++);                            // the first (no values before it) ...
#pragma unroll 1
        while (t < whole) step(WholeTile(), t++);
    }                                                    // ... and those at the end
    if (n > 0 && (t0 + n - 1) * KT2 < wave_max) {
        values(n - 1);
        if (partial_tile(n - 1)) values_not_finite(n - 1);
    }
    if (!half) __syncthreads();                          // (half 1's last vector phase)

    auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    const float L = __uint_as_float(w[0]) + __uint_as_float(w[1]);
    if (!on) return;
    if (a.parts == 1) {
        const float inv = inverse_sum(L, seen > 0);
        bf16_t* op = a.out + (size_t)token * a.ldo + head * HD + 4 * h;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *(uint2*)(op + 32 * i + 8 * e) = make_uint2(pack2bf(o[i][4 * e] * inv, o[i][4 * e + 1] * inv), pack2bf(o[i][4 * e + 2] * inv, o[i][4 * e + 3] * inv));
    } else {
        const long long at = (long long)(p.part0 + split) * a.rows + (long long)token * a.H + head;
        if (L != 0.f) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    *(f32x4*)(a.o_part + at * HD + 32 * i + 8 * e + 4 * h) = (f32x4){o[i][4 * e], o[i][4 * e + 1], o[i][4 * e + 2], o[i][4 * e + 3]};
        }
        if (h == 0) a.ml_part[at] = make_float2(m == -INFINITY ? LOWEST : -nref, L);
    }
}

// The parts of every row joined.  Thread = 4 channels of a row and every JW-th of its parts (few rows have many parts: a thread that walked
// them all would wait for one memory round trip after the other); the JW partial sums meet in the LDS.  JW = 8 from five parts on (48 slots
// behind a prefix, 33 parts: 61 us in all against 72 with 1), 1 below (64 K rows of two parts: 110 us in all against 136 with 8).
struct JoinSees { const int* kv_lens; int kv_len, rows, T, causal, prefix; };              // what rows_of_slot takes; with a prefix every row sees keys
template <int HD, int JW>
__global__ __launch_bounds__(256) void kv_attention_join_kernel(const float* __restrict__ o_part, const float2* __restrict__ ml, long long rows,
                                                                int parts, int H, bf16_t* __restrict__ out, int ldo, const JoinSees v) {
    constexpr int LPR = HD / 4, RPB = 256 / (LPR * JW);  // threads of a row's channels, rows of a workgroup
    const int c = threadIdx.x % LPR, w = (threadIdx.x / LPR) % JW, lr = threadIdx.x / (LPR * JW);
    const long long row = (long long)blockIdx.x * RPB + lr;
    const bool on = row < rows;
    float M = LOWEST, L = 0.f;
    f32x4 o = (f32x4){0.f, 0.f, 0.f, 0.f};
    if (on) {
#pragma unroll 4
        for (int p = w; p < parts; p += JW) {
            const float2 x = ml[p * rows + row];
            if (x.y != 0.f) join_part(M, L, o, x.x, x.y, *(const f32x4*)(o_part + (p * rows + row) * HD + 4 * c));
        }
    }
    if (JW > 1) {
        __shared__ f32x4 so[JW > 1 ? 256 : 1];
        __shared__ float2 sl[JW > 1 ? 256 : 1];
        so[threadIdx.x] = o;
        sl[threadIdx.x] = make_float2(M, L);
        __syncthreads();
        if (w || !on) return;
#pragma unroll
        for (int k = 1; k < JW; ++k) join_part(M, L, o, sl[threadIdx.x + k * LPR].x, sl[threadIdx.x + k * LPR].y, so[threadIdx.x + k * LPR]);
    }
    if (!on) return;
    const int token = (int)(row / H);
    bool sees = v.prefix != 0;
    if (L == 0.f && !sees) {
        const int n = rows_of_slot(v.kv_lens, v.kv_len, v.rows, token / v.T);
        sees = (v.causal ? n - v.T + token % v.T + 1 : n) > 0;
    }
    store_row_quad(out + (size_t)token * ldo + (row % H) * HD + 4 * c, L, sees, o);
}

__global__ void kv_zero_kernel(unsigned* p, int n) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) p[i] = 0u;
}

// ------------------------------------------------------------------------------------------------ host side
int check_cache(const char* who, const seedmi_kv_cache_t* c, KvView* v) {
    if (!c || !c->k || !c->v || c->slots <= 0 || c->rows <= 0 || c->kv_heads <= 0 || c->head_rows < 0 || c->slot_rows < 0) {
        seedmi_set_error("%s: cache handle: null pointer or slots / rows / kv_heads <= 0 or a negative stride", who);
        return SEEDMI_E_SHAPE;
    }
    if (c->rows > 1 << 22) {                               // (32-bit offsets inside a (slot, head))
        seedmi_set_error("%s: %d rows (at most 2^22)", who, c->rows);
        return SEEDMI_E_SHAPE;
    }
    if (c->head_dim != 64 && c->head_dim != 128) {
        seedmi_set_error("%s: head_dim %d (must be 64 or 128)", who, c->head_dim);
        return SEEDMI_E_SHAPE;
    }
    if (c->format != SEEDMI_KV_16BIT && c->format != SEEDMI_KV_MX8) {
        seedmi_set_error("%s: cache format %d (SEEDMI_KV_16BIT or SEEDMI_KV_MX8)", who, c->format);
        return SEEDMI_E_DTYPE;
    }
    const bool mx = c->format == SEEDMI_KV_MX8;
    if (mx != (c->k_scale != nullptr) || mx != (c->v_scale != nullptr)) {
        seedmi_set_error("%s: scale bytes belong to an MX8 cache and to no other", who);
        return SEEDMI_E_SHAPE;
    }
    if ((((uintptr_t)c->k | (uintptr_t)c->v) & 15) || (((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & (unsigned)(c->head_dim / 32 - 1))) {
        seedmi_set_error("%s: k / v must be 16-byte aligned, k_scale / v_scale aligned to a row's head_dim / 32 bytes", who);
        return SEEDMI_E_ALIGN;
    }
    *v = {(char*)c->k, (char*)c->v, (uint8_t*)c->k_scale, (uint8_t*)c->v_scale, c->slot_rows, c->head_rows, c->rows, c->kv_heads};
    return SEEDMI_OK;
}

}  // namespace

#define KV_DISPATCH(hd, mx, CALL)                                      \
    do {                                                               \
        if ((hd) == 128) { if (mx) { CALL(128, true); } else { CALL(128, false); } } \
        else { if (mx) { CALL(64, true); } else { CALL(64, false); } }  \
    } while (0)

// seedmi_kv_append / seedmi_kv_attention, or their checks alone (launch == false): a path of many launches refuses before the first one
int seedmi_kv_append_impl(const seedmi_kv_cache_t* cache, const void* qkv, int ldqkv, const void* pos_ids_i64, int pos_base, const void* cos_t,
                          const void* sin_t, int max_pos, void* q_out, int ldq, int B, int T, int H, int past_len, const void* past_lens_i32,
                          void* stream, bool launch) {
    KvView v;
    if (const int rc = check_cache("seedmi_kv_append", cache, &v)) return rc;
    const int hd = cache->head_dim, G = cache->kv_heads;
    if (!qkv || !cos_t || !sin_t || !q_out || B <= 0 || B > cache->slots || T <= 0 || H <= 0 || max_pos <= 0 || pos_base < 0 ||
        ldqkv < (long long)(H + 2ll * G) * hd || ldq < (long long)H * hd) {
        seedmi_set_error("seedmi_kv_append: null pointer or bad shape: B=%d (slots %d) T=%d H=%d kv_heads=%d ldqkv=%d ldq=%d max_pos=%d", B,
                         cache->slots, T, H, G, ldqkv, ldq, max_pos);
        return SEEDMI_E_SHAPE;
    }
    const bool by_slot = (B == 1 || v.slot_rows >= (G - 1) * v.head_rows + v.rows) && (G == 1 || v.head_rows >= v.rows);
    const bool by_head = (G == 1 || v.head_rows >= (B - 1) * v.slot_rows + v.rows) && (B == 1 || v.slot_rows >= v.rows);
    if (!by_slot && !by_head) {
        seedmi_set_error("seedmi_kv_append: rows of different slots / heads overlap (slot_rows %lld, head_rows %lld, rows %d)", v.slot_rows,
                         v.head_rows, v.rows);
        return SEEDMI_E_SHAPE;
    }
    if (!past_lens_i32 && (past_len < 0 || (long long)past_len + T > cache->rows)) {
        seedmi_set_error("seedmi_kv_append: rows %d .. %lld of a cache of %d", past_len, (long long)past_len + T - 1, cache->rows);
        return SEEDMI_E_SHAPE;
    }
    if ((ldqkv % 8) || (ldq % 8) || (((uintptr_t)qkv | (uintptr_t)cos_t | (uintptr_t)sin_t | (uintptr_t)q_out) & 15) ||
        ((uintptr_t)pos_ids_i64 & 7) || ((uintptr_t)past_lens_i32 & 3)) {
        seedmi_set_error("seedmi_kv_append: pointers 16-byte aligned, leading dimensions multiples of 8");
        return SEEDMI_E_ALIGN;
    }
    const long long total = (long long)B * T * (H + 2ll * G) * (hd / 16);
    if (total > INT_MAX) {
        seedmi_set_error("seedmi_kv_append: B * T * (H + 2 kv_heads) * head_dim / 16 = %lld: at most 2^31 - 1", total);
        return SEEDMI_E_SHAPE;
    }
    if (!launch) return SEEDMI_OK;
#define CALL(HD, MX)                                                                                                                         \
    hipLaunchKernelGGL((kv_append_kernel<HD, MX>), dim3((unsigned)((total + 255) / 256)), dim3(256), 0, (hipStream_t)stream, v,              \
                       (const bf16_t*)qkv, ldqkv, (const long long*)pos_ids_i64, pos_base, (const bf16_t*)cos_t, (const bf16_t*)sin_t,       \
                       max_pos, (bf16_t*)q_out, ldq, B, T, H, past_len, (const int*)past_lens_i32)
    KV_DISPATCH(hd, cache->format == SEEDMI_KV_MX8, CALL);
#undef CALL
    return seedmi_check_launch("kv_append");
}

extern "C" int seedmi_kv_append(const seedmi_kv_cache_t* cache, const void* qkv, int ldqkv, const void* pos_ids_i64, int pos_base,
                                const void* cos_t, const void* sin_t, int max_pos, void* q_out, int ldq, int B, int T, int H, int past_len,
                                const void* past_lens_i32, void* stream) {
    return seedmi_kv_append_impl(cache, qkv, ldqkv, pos_ids_i64, pos_base, cos_t, sin_t, max_pos, q_out, ldq, B, T, H, past_len, past_lens_i32,
                                 stream, true);
}

extern "C" int seedmi_kv_read(const seedmi_kv_cache_t* cache, void* k_out, void* v_out, int B, int n, int start, const void* starts_i32,
                              void* stream) {
    KvView v;
    if (const int rc = check_cache("seedmi_kv_read", cache, &v)) return rc;
    if (cache->format != SEEDMI_KV_MX8) {
        seedmi_set_error("seedmi_kv_read: the rows of a 16-bit cache are what they are: only MX8 caches are read back");
        return SEEDMI_E_DTYPE;
    }
    if ((n > 0 && !k_out && !v_out) || B <= 0 || B > cache->slots || n < 0 || (!starts_i32 && (start < 0 || (long long)start + n > cache->rows))) {
        seedmi_set_error("seedmi_kv_read: no output, B=%d (slots %d), or rows %d .. + %d of a cache of %d", B, cache->slots, start, n, cache->rows);
        return SEEDMI_E_SHAPE;
    }
    if ((((uintptr_t)k_out | (uintptr_t)v_out) & 15) || ((uintptr_t)starts_i32 & 3)) {
        seedmi_set_error("seedmi_kv_read: outputs must be 16-byte aligned");
        return SEEDMI_E_ALIGN;
    }
    if (n == 0) return SEEDMI_OK;
    const long long total = (long long)B * cache->kv_heads * n * (cache->head_dim / 16);
    const long long blocks = (total + 255) / 256;
    const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)), (k_out && v_out) ? 2 : 1);
    if (cache->head_dim == 128)
        hipLaunchKernelGGL(kv_read_kernel<128>, grid, dim3(256), 0, (hipStream_t)stream, v, (bf16_t*)k_out, (bf16_t*)v_out, B, n, start, (const int*)starts_i32);
    else
        hipLaunchKernelGGL(kv_read_kernel<64>, grid, dim3(256), 0, (hipStream_t)stream, v, (bf16_t*)k_out, (bf16_t*)v_out, B, n, start, (const int*)starts_i32);
    return seedmi_check_launch("kv_read");
}

// How a call is cut: a pass over the slots' own rows and, with a prefix, one over the prefix; row blocks and key ranges of each.
struct KvPass { int groups, group_rows, block_rows, row_blocks, splits, per_split; long long blocks; };
struct KvPlan {
    KvPass own, pre;
    int parts, units, unit_rows;                         // units > 0: joined in place, by the last workgroup of each unit
    unsigned unit_blocks;
    long long rows;
    size_t bytes, o_at;                                  // workspace: arrival counters, (m, l) from KV_WS_COUNTERS on, sums from o_at on
};
constexpr size_t KV_WS_COUNTERS = 4096;                  // bytes: 1024 counters

static KvPass plan_pass(int groups, long long rows, long long keys) {
    KvPass p = {};
    p.groups = groups;
    p.group_rows = (int)rows;
    // Rows of a block: the smallest that holds the group.  us for 8 x 40 heads x 1024 past rows, 8-bit, by the rows of a group (column: block):
    //   rows    16    32    64   128   256        (16-bit rows: the same order, 33 - 37 us up to 64 rows)
    //     16  21.6  22.8  27.0  33.8  50.7
    //     32  25.8  24.5  31.8  35.4  51.6
    //     48  32.0  34.4  34.1  44.5  53.9
    //    100        51.4  57.6  53.5  60.1        2 x 8 heads x 8000 past rows, 96 rows: 24.5  26.7  26.5  24.2
    //    256             100.3  93.0  93.1                                          192 rows:       37.1  37.3  33.3
    // More than 256 rows leave a block of them partly empty; where that costs a round of workgroups in five, blocks of 128 (two to a CU):
    // 300 rows of 320 groups 110 us against 134, of 16 groups 50 against 44.
    p.block_rows = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
    if (p.block_rows == 256) {
        const long long by256 = ((rows + 255) / 256 * groups + 255) / 256, by128 = ((rows + 127) / 128 * groups + 511) / 512;
        if (by128 * 5 < by256 * 4) p.block_rows = 128;
    }
    p.row_blocks = (int)((rows + p.block_rows - 1) / p.block_rows);
    const int kt = p.block_rows <= 32 ? KT : KT2;
    const long long tiles = (keys + kt - 1) / kt, base = (long long)groups * p.row_blocks;
    // One workgroup per CU, two of the 64- and 128-row ones (they share a CU).  Few rows: between 256 and 2048 workgroups it is flat within
    // the noise for 4 slots of up to 65 thousand rows (82 - 85 us) and slower from 2048 on for 32 slots (68 -> 73).  192 rows of 48 slots
    // behind a prefix of 24 thousand: 62 us in 256-row blocks (75 with 128 workgroups), 76 -> 69 in 128-row ones and 79 -> 65 in 64-row ones
    // from 256 to 512 workgroups.
    // At least four tiles to a range (a tile per wave): one conversation 8.35 us, with two 8.76, with eight 8.88.  A range has a fixed number
    // of tiles (of the longest slot expected), so short slots have fewer; the slots take turns from range to range, so that the CUs get as
    // many of them each.
    const long long target = p.block_rows == 64 || p.block_rows == 128 ? 512 : 256;
    long long s = target / base;
    if (s > (tiles + MIN_TILES - 1) / MIN_TILES) s = (tiles + MIN_TILES - 1) / MIN_TILES;
    p.splits = (int)(s < 1 ? 1 : s);
    p.per_split = (int)((tiles + p.splits - 1) / p.splits);
    if (p.per_split < MIN_TILES) p.per_split = MIN_TILES;
    p.blocks = ((long long)p.groups * p.splits + 7) / 8 * 8 * p.row_blocks;
    return p;
}

// 0: fits; -1: not a shape the kernels take (the callers have checked pointers)
static int make_plan(const seedmi_kv_cache_t* c, int B, int T, int H, int kv_max, int prefix_len, KvPlan* pl) {
    if (!c || c->slots <= 0 || c->rows <= 0 || c->kv_heads <= 0 || B <= 0 || B > c->slots || T <= 0 || H <= 0 || H % c->kv_heads || kv_max < 0 ||
        prefix_len < 0)
        return -1;
    pl->rows = (long long)B * T * H;
    if (pl->rows > INT_MAX) return -1;
    const int GH = H / c->kv_heads;
    const long long keys = kv_max == 0 || kv_max > c->rows ? c->rows : kv_max;
    if ((long long)B * c->kv_heads > INT_MAX / 64) return -1;
    pl->own = plan_pass(B * c->kv_heads, (long long)T * GH, keys);
    pl->pre = prefix_len ? plan_pass(c->kv_heads, (long long)B * T * GH, prefix_len) : KvPass{};
    pl->parts = pl->own.splits + pl->pre.splits;
    // a launch has fewer than 2^32 threads
    if ((pl->own.blocks + pl->pre.blocks) * 512 > UINT_MAX || (pl->parts > 1 && pl->rows * (c->head_dim / 4) * 8 > UINT_MAX)) return -1;
    pl->units = pl->unit_rows = 0;
    pl->unit_blocks = 0;
    if (pl->parts > 1 && pl->own.block_rows <= 32 && (!prefix_len || pl->pre.block_rows == pl->own.block_rows)) {
        // Joined in place where a unit's rows and parts are few enough for one workgroup: a second launch costs about 3 us (one conversation
        // of 700 rows 8.1 against 11.4 us, four samples behind a prompt 10.5 against 11.6)
        const int rows = prefix_len ? pl->pre.group_rows : pl->own.block_rows < pl->own.group_rows ? pl->own.block_rows : pl->own.group_rows;
        const long long units = prefix_len ? c->kv_heads : (long long)pl->own.groups * pl->own.row_blocks;
        if ((long long)rows * pl->parts <= 64 && units * 4 <= (long long)KV_WS_COUNTERS) {
            pl->units = (int)units;
            pl->unit_rows = prefix_len ? rows : 0;
            pl->unit_blocks = prefix_len ? (unsigned)(pl->pre.row_blocks * pl->pre.splits + B * pl->own.row_blocks * pl->own.splits) : (unsigned)pl->own.splits;
        }
    }
    pl->o_at = (KV_WS_COUNTERS + (size_t)pl->parts * pl->rows * 8 + 255) & ~(size_t)255;
    pl->bytes = pl->parts == 1 ? 0 : pl->o_at + (size_t)pl->parts * pl->rows * c->head_dim * 4;
    return 0;
}

extern "C" size_t seedmi_kv_attention_workspace_bytes(const seedmi_kv_cache_t* cache, int B, int T, int H, int kv_max, int prefix_len) {
    KvPlan pl;
    return make_plan(cache, B, T, H, kv_max, prefix_len, &pl) ? 0 : pl.bytes;
}

extern "C" int seedmi_kv_attention_workspace_init(void* workspace, size_t workspace_bytes, void* stream) {
    if (workspace_bytes == 0) return SEEDMI_OK;
    if (!workspace || workspace_bytes < KV_WS_COUNTERS || ((uintptr_t)workspace & 255)) {
        seedmi_set_error("seedmi_kv_attention_workspace_init: need seedmi_kv_attention_workspace_bytes() bytes, 256-byte aligned");
        return SEEDMI_E_ALIGN;
    }
    hipLaunchKernelGGL(kv_zero_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream, (unsigned*)workspace, (int)(KV_WS_COUNTERS / 4));
    return seedmi_check_launch("kv_attention_workspace_init");
}

template <int HD, bool MX>
static void launch_blocks(const AttnArgs& a, int block_rows, unsigned blocks, hipStream_t s) {
    switch (block_rows) {
        case 16: hipLaunchKernelGGL((kv_attention_few_kernel<HD, MX, 1>), dim3(blocks), dim3(256), 0, s, a); break;
        case 32: hipLaunchKernelGGL((kv_attention_few_kernel<HD, MX, 2>), dim3(blocks), dim3(256), 0, s, a); break;
        case 64: hipLaunchKernelGGL((kv_attention_many_kernel<HD, MX, 1>), dim3(blocks), dim3(256), 0, s, a); break;
        case 128: hipLaunchKernelGGL((kv_attention_many_kernel<HD, MX, 2>), dim3(blocks), dim3(256), 0, s, a); break;
        default: hipLaunchKernelGGL((kv_attention_phased_kernel<HD, MX>), dim3(blocks), dim3(512), 0, s, a); break;
    }
}

template <int HD, int JW>
static void launch_join(const AttnArgs& a, const KvPlan& pl, const JoinSees& v, hipStream_t s) {
    constexpr int RPB = 256 / (HD / 4 * JW);
    hipLaunchKernelGGL((kv_attention_join_kernel<HD, JW>), dim3((unsigned)((pl.rows + RPB - 1) / RPB)), dim3(256), 0, s, a.o_part, a.ml_part,
                       pl.rows, pl.parts, a.H, a.out, a.ldo, v);
}

template <int HD, bool MX>
static void launch_attention(AttnArgs a, const KvView& own, const KvView& pre, const KvPlan& pl, int prefix_len, int kv_len, const int* kv_lens,
                             hipStream_t s) {
    auto set = [](AttnPass& x, const KvView& v, const KvPass& p, int shared, int part0, int len, const int* lens) {
        x = {v, lens, len, shared, p.groups, p.group_rows, p.row_blocks, p.splits, part0, p.per_split, (unsigned)p.blocks};
    };
    if (!prefix_len) {
        set(a.pass[0], own, pl.own, 0, 0, kv_len, kv_lens);
        launch_blocks<HD, MX>(a, pl.own.block_rows, (unsigned)pl.own.blocks, s);
    } else {
        set(a.pass[0], pre, pl.pre, 1, 0, prefix_len, nullptr);
        set(a.pass[1], own, pl.own, 0, pl.pre.splits, kv_len, kv_lens);
        if (pl.pre.block_rows == pl.own.block_rows) {    // one kernel for both: one launch
            launch_blocks<HD, MX>(a, pl.own.block_rows, (unsigned)(pl.pre.blocks + pl.own.blocks), s);
        } else {
            launch_blocks<HD, MX>(a, pl.pre.block_rows, (unsigned)pl.pre.blocks, s);
            a.pass[0] = a.pass[1];
            launch_blocks<HD, MX>(a, pl.own.block_rows, (unsigned)pl.own.blocks, s);
        }
    }
    if (pl.parts > 1 && !pl.units) {
        const JoinSees v = {kv_lens, kv_len, own.rows, a.T, a.causal, prefix_len};
        if (pl.parts > 4) launch_join<HD, 8>(a, pl, v, s);
        else launch_join<HD, 1>(a, pl, v, s);
    }
}

constexpr float LOG2E = 1.44269504088896340736f;

int seedmi_kv_attention_impl(const seedmi_kv_cache_t* cache, const seedmi_kv_cache_t* prefix, int prefix_len, const void* q, int ldq, void* out,
                             int ldo, int B, int T, int H, int kv_len, const void* kv_lens_i32, int kv_max, float scale, int causal,
                             void* workspace, size_t workspace_bytes, void* stream, bool launch) {
    KvView own, pre;
    if (const int rc = check_cache("seedmi_kv_attention", cache, &own)) return rc;
    const int hd = cache->head_dim, G = cache->kv_heads;
    if (prefix_len < 0 || (prefix_len > 0 && !prefix)) {
        seedmi_set_error("seedmi_kv_attention: prefix_len %d without a prefix", prefix_len);
        return SEEDMI_E_SHAPE;
    }
    pre = own;
    if (prefix_len) {
        if (const int rc = check_cache("seedmi_kv_attention (prefix)", prefix, &pre)) return rc;
        if (prefix->head_dim != hd || prefix->kv_heads != G || prefix->format != cache->format || prefix_len > prefix->rows) {
            seedmi_set_error("seedmi_kv_attention: the prefix has head_dim %d, %d key heads, format %d, %d rows (%d asked); the cache %d, %d, %d",
                             prefix->head_dim, prefix->kv_heads, prefix->format, prefix->rows, prefix_len, hd, G, cache->format);
            return SEEDMI_E_SHAPE;
        }
    }
    if (!q || !out || B <= 0 || B > cache->slots || T <= 0 || H <= 0 || (H % G) || ldq < (long long)H * hd || ldo < (long long)H * hd ||
        kv_max < 0 || !(scale > 0.f) || !(scale * LOG2E <= FLT_MAX)) {
        seedmi_set_error("seedmi_kv_attention: null pointer or bad shape: B=%d (slots %d) T=%d H=%d (a multiple of %d) ldq=%d ldo=%d kv_max=%d "
                         "scale=%g (above 0, finite in base-2 exponents: at most 2.3e38)", B, cache->slots, T, H, G, ldq, ldo, kv_max, scale);
        return SEEDMI_E_SHAPE;
    }
    if (kv_len < 0 || kv_len > cache->rows) {
        seedmi_set_error("seedmi_kv_attention: kv_len %d of a cache of %d rows", kv_len, cache->rows);
        return SEEDMI_E_SHAPE;
    }
    if ((ldq % 8) || (ldo % 8) || (((uintptr_t)q | (uintptr_t)out) & 15) || ((uintptr_t)kv_lens_i32 & 3)) {
        seedmi_set_error("seedmi_kv_attention: pointers 16-byte aligned, leading dimensions multiples of 8");
        return SEEDMI_E_ALIGN;
    }
    KvPlan pl;
    if (make_plan(cache, B, T, H, kv_max, prefix_len, &pl)) {
        seedmi_set_error("seedmi_kv_attention: B * T * H = %lld rows need more threads than a launch has (2^32)", (long long)B * T * H);
        return SEEDMI_E_SHAPE;
    }
    if (pl.bytes && (!workspace || workspace_bytes < pl.bytes || ((uintptr_t)workspace & 255))) {
        seedmi_set_error("seedmi_kv_attention: workspace %zu bytes (need %zu, 256-byte aligned)", workspace_bytes, pl.bytes);
        return SEEDMI_E_ALIGN;
    }
    if (!launch) return SEEDMI_OK;
    AttnArgs a = {};
    a.q = (const bf16_t*)q;
    a.out = (bf16_t*)out;
    a.ldq = ldq; a.ldo = ldo; a.T = T; a.H = H; a.GH = H / G;
    a.causal = causal; a.c2 = scale * LOG2E;
    a.rows = pl.rows; a.parts = pl.parts;
    a.arrivals = pl.units ? (unsigned*)workspace : nullptr;
    a.unit_blocks = pl.unit_blocks; a.unit_rows = pl.unit_rows;
    a.ml_part = (float2*)((char*)workspace + KV_WS_COUNTERS);
    a.o_part = (float*)((char*)workspace + pl.o_at);
#define CALL(HD, MX) launch_attention<HD, MX>(a, own, pre, pl, prefix_len, kv_len, (const int*)kv_lens_i32, (hipStream_t)stream)
    KV_DISPATCH(hd, cache->format == SEEDMI_KV_MX8, CALL);
#undef CALL
    return seedmi_check_launch("kv_attention");
}

extern "C" int seedmi_kv_attention(const seedmi_kv_cache_t* cache, const seedmi_kv_cache_t* prefix, int prefix_len, const void* q, int ldq,
                                   void* out, int ldo, int B, int T, int H, int kv_len, const void* kv_lens_i32, int kv_max, float scale,
                                   int causal, void* workspace, size_t workspace_bytes, void* stream) {
    return seedmi_kv_attention_impl(cache, prefix, prefix_len, q, ldq, out, ldo, B, T, H, kv_len, kv_lens_i32, kv_max, scale, causal, workspace,
                                    workspace_bytes, stream, true);
}
