// KV cache by handle (include/seedmi.h: seedmi_kv_cache_t): rows written, read back and attended to.
//
//  seedmi_kv_append     apply_rotary_pos_emb + append (llama_xformer.py:160-168, 234-239) into 16-bit or 8-bit rows, grouped heads, one
//                       length per slot
//  seedmi_kv_read       8-bit rows back as 16-bit tensors
//  seedmi_kv_attention  memory_efficient_attention over the cache (llama_xformer.py:244-256), optionally behind a prefix that all slots share
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
// One thread = 8 values i .. i + 7 and their partners i + HD/2 .. of one (slot, token, head): a quad of lanes holds two whole blocks of 32.
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
// One thread = 16 values: 16 code bytes in, 32 bytes out.  blockIdx.y: keys / values.
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
struct AttnArgs {
    KvView c, p;                                         // the slots' cache, the shared prefix
    const bf16_t* q;
    bf16_t* out;
    int ldq, ldo, B, T, H, kv_len, prefix_len, causal;
    const int* kv_lens;
    float scale;
};

// One wave = one query row: lane = HD / 64 values of the row, keys one after the other.
template <int HD, bool MX>
__global__ __launch_bounds__(256) void kv_attention_rows_kernel(const AttnArgs a) {
    constexpr int VPL = HD / 64;
    const int lane = threadIdx.x & 63;
    const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= (long long)a.B * a.T * a.H) return;
    const int h = (int)(r % a.H);
    const int row = (int)(r / a.H);
    const int b = row / a.T, t = row - b * a.T;
    const int g = h / (a.H / a.c.G);
    const int len = max(0, min(a.kv_lens ? a.kv_lens[b] : a.kv_len, a.c.rows));
    const int seen = a.causal ? max(0, len - a.T + t + 1) : len;
    float q[VPL], o[VPL], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
        q[v] = bf2f(a.q[(size_t)row * a.ldq + h * HD + lane * VPL + v]) * a.scale;
        o[v] = 0.f;
    }
    auto val = [&](const char* base, const uint8_t* sc, long long crow, int v) -> float {
        const int d = lane * VPL + v;
        if (!MX) return bf2f(((const bf16_t*)base)[crow * HD + d]);
        const uint32_t w = mx_unpack2<false>((uint32_t)(uint8_t)base[crow * HD + d], mx_scale_f(sc[crow * (HD / 32) + d / 32]));
        return lo_bf(w);
    };
    auto walk = [&](const KvView& c, long long first, int n) {
        for (int j = 0; j < n; ++j) {
            float s = 0.f;
#pragma unroll
            for (int v = 0; v < VPL; ++v) s += q[v] * val(c.k, c.ks, first + j, v);
            s = wave_sum(s);
            const float mn = fmaxf(m, s);
            const float f = __expf(m - mn), p = __expf(s - mn);
            l = l * f + p;
            m = mn;
#pragma unroll
            for (int v = 0; v < VPL; ++v) o[v] = o[v] * f + p * val(c.v, c.vs, first + j, v);
        }
    };
    if (a.prefix_len) walk(a.p, (long long)g * a.p.head_rows, a.prefix_len);
    walk(a.c, (long long)b * a.c.slot_rows + (long long)g * a.c.head_rows, seen);
#pragma unroll
    for (int v = 0; v < VPL; ++v)
        a.out[(size_t)row * a.ldo + h * HD + lane * VPL + v] = f2bf(l == 0.f ? 0.f : o[v] / l);
}

// ------------------------------------------------------------------------------------------------ host side
int check_cache(const char* who, const seedmi_kv_cache_t* c, KvView* v) {
    if (!c || !c->k || !c->v || c->slots <= 0 || c->rows <= 0 || c->kv_heads <= 0 || c->head_rows < 0 || c->slot_rows < 0) {
        seedmi_set_error("%s: cache handle: null pointer or slots / rows / kv_heads <= 0 or a negative stride", who);
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
    if ((((uintptr_t)c->k | (uintptr_t)c->v) & 15) || (((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 3)) {
        seedmi_set_error("%s: k / v must be 16-byte aligned, k_scale / v_scale 4-byte aligned", who);
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

extern "C" int seedmi_kv_append(const seedmi_kv_cache_t* cache, const void* qkv, int ldqkv, const void* pos_ids_i64, int pos_base,
                                const void* cos_t, const void* sin_t, int max_pos, void* q_out, int ldq, int B, int T, int H, int past_len,
                                const void* past_lens_i32, void* stream) {
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
#define CALL(HD, MX)                                                                                                                         \
    hipLaunchKernelGGL((kv_append_kernel<HD, MX>), dim3((unsigned)((total + 255) / 256)), dim3(256), 0, (hipStream_t)stream, v,              \
                       (const bf16_t*)qkv, ldqkv, (const long long*)pos_ids_i64, pos_base, (const bf16_t*)cos_t, (const bf16_t*)sin_t,       \
                       max_pos, (bf16_t*)q_out, ldq, B, T, H, past_len, (const int*)past_lens_i32)
    KV_DISPATCH(hd, cache->format == SEEDMI_KV_MX8, CALL);
#undef CALL
    return seedmi_check_launch("kv_append");
}

extern "C" int seedmi_kv_read(const seedmi_kv_cache_t* cache, void* k_out, void* v_out, int B, int n, int start, const void* starts_i32,
                              void* stream) {
    KvView v;
    if (const int rc = check_cache("seedmi_kv_read", cache, &v)) return rc;
    if (cache->format != SEEDMI_KV_MX8) {
        seedmi_set_error("seedmi_kv_read: the rows of a 16-bit cache are what they are: only MX8 caches are read back");
        return SEEDMI_E_DTYPE;
    }
    if ((!k_out && !v_out) || B <= 0 || B > cache->slots || n < 0 || (!starts_i32 && (start < 0 || (long long)start + n > cache->rows))) {
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

extern "C" size_t seedmi_kv_attention_workspace_bytes(const seedmi_kv_cache_t* cache, int B, int T, int H, int kv_max, int prefix_len) {
    (void)cache; (void)B; (void)T; (void)H; (void)kv_max; (void)prefix_len;
    return 0;
}

extern "C" int seedmi_kv_attention(const seedmi_kv_cache_t* cache, const seedmi_kv_cache_t* prefix, int prefix_len, const void* q, int ldq,
                                   void* out, int ldo, int B, int T, int H, int kv_len, const void* kv_lens_i32, int kv_max, float scale,
                                   int causal, void* workspace, size_t workspace_bytes, void* stream) {
    AttnArgs a = {};
    if (const int rc = check_cache("seedmi_kv_attention", cache, &a.c)) return rc;
    const int hd = cache->head_dim, G = cache->kv_heads;
    if (prefix_len < 0 || (prefix_len > 0 && !prefix)) {
        seedmi_set_error("seedmi_kv_attention: prefix_len %d without a prefix", prefix_len);
        return SEEDMI_E_SHAPE;
    }
    a.p = a.c;
    if (prefix_len) {
        if (const int rc = check_cache("seedmi_kv_attention (prefix)", prefix, &a.p)) return rc;
        if (prefix->head_dim != hd || prefix->kv_heads != G || prefix->format != cache->format || prefix_len > prefix->rows) {
            seedmi_set_error("seedmi_kv_attention: the prefix has head_dim %d, %d key heads, format %d, %d rows (%d asked); the cache %d, %d, %d",
                             prefix->head_dim, prefix->kv_heads, prefix->format, prefix->rows, prefix_len, hd, G, cache->format);
            return SEEDMI_E_SHAPE;
        }
    }
    if (!q || !out || B <= 0 || B > cache->slots || T <= 0 || H <= 0 || (H % G) || ldq < (long long)H * hd || ldo < (long long)H * hd ||
        kv_max < 0 || !(scale == scale)) {
        seedmi_set_error("seedmi_kv_attention: null pointer or bad shape: B=%d (slots %d) T=%d H=%d (a multiple of %d) ldq=%d ldo=%d kv_max=%d", B,
                         cache->slots, T, H, G, ldq, ldo, kv_max);
        return SEEDMI_E_SHAPE;
    }
    if (!kv_lens_i32 && (kv_len < 0 || kv_len > cache->rows)) {
        seedmi_set_error("seedmi_kv_attention: kv_len %d of a cache of %d rows", kv_len, cache->rows);
        return SEEDMI_E_SHAPE;
    }
    if ((ldq % 8) || (ldo % 8) || (((uintptr_t)q | (uintptr_t)out) & 15) || ((uintptr_t)kv_lens_i32 & 3)) {
        seedmi_set_error("seedmi_kv_attention: pointers 16-byte aligned, leading dimensions multiples of 8");
        return SEEDMI_E_ALIGN;
    }
    const long long rows = (long long)B * T * H;
    if (rows > INT_MAX) {
        seedmi_set_error("seedmi_kv_attention: B * T * H = %lld: at most 2^31 - 1", rows);
        return SEEDMI_E_SHAPE;
    }
    const size_t need = seedmi_kv_attention_workspace_bytes(cache, B, T, H, kv_max, prefix_len);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255))) {
        seedmi_set_error("seedmi_kv_attention: workspace %zu bytes (need %zu, 256-byte aligned)", workspace_bytes, need);
        return SEEDMI_E_ALIGN;
    }
    a.q = (const bf16_t*)q; a.out = (bf16_t*)out;
    a.ldq = ldq; a.ldo = ldo; a.B = B; a.T = T; a.H = H;
    a.kv_len = kv_len; a.kv_lens = (const int*)kv_lens_i32;
    a.prefix_len = prefix_len; a.causal = causal; a.scale = scale;
#define CALL(HD, MX)                                                                                                            \
    hipLaunchKernelGGL((kv_attention_rows_kernel<HD, MX>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, (hipStream_t)stream, a)
    KV_DISPATCH(hd, cache->format == SEEDMI_KV_MX8, CALL);
#undef CALL
    return seedmi_check_launch("kv_attention");
}
