// Key / value cache in 8 bits and the attention over it, gfx950 (CDNA4, wave64).  Format: include/acmi.h (acmi_kv8_cache).
// Reference semantics: audiocraft/modules/transformer.py:266-298 (_complete_kv), :412-414 (scaled_dot_product_attention).
#include "acmi_lm_internal.h"

#include <math.h>

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float kv8_f32x2 __attribute__((ext_vector_type(2)));

constexpr int BLK = ACMI_KV8_BLOCK;

__device__ __forceinline__ float kv8_ld(const void* p, size_t i, int bf16) {
    return bf16 ? bf16_to_f32(reinterpret_cast<const bf16_t*>(p)[i]) : reinterpret_cast<const float*>(p)[i];
}
__device__ __forceinline__ void kv8_st(void* p, size_t i, int bf16, float v) {
    if (bf16) reinterpret_cast<bf16_t*>(p)[i] = f32_to_bf16(v);
    else reinterpret_cast<float*>(p)[i] = v;
}
// what the tail makes of a value
__device__ __forceinline__ float kv8_round(float v, int bf16) { return bf16 ? bf16_to_f32(f32_to_bf16(v)) : v; }

// maximum over the four lanes of a column (xor 16, xor 32) without the LDS crossbar: a swap of a register with its own copy leaves
// the two halves of every pair side by side
__device__ __forceinline__ float kv8_xmax(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// 16 consecutive features (16-byte aligned) -> f32
__device__ __forceinline__ void kv8_ld16(const void* p, size_t i, int bf16, float (&x)[16]) {
    if (bf16) {
        const u32x4* q = reinterpret_cast<const u32x4*>(reinterpret_cast<const bf16_t*>(p) + i);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const u32x4 w = q[h];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[h * 8 + e * 2] = __uint_as_float(w[e] << 16);
                x[h * 8 + e * 2 + 1] = __uint_as_float(w[e] & 0xffff0000u);
            }
        }
    } else {
        const f32x4* q = reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(p) + i);
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            const f32x4 w = q[h];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[h * 4 + e] = w[e];
        }
    }
}
// 4 consecutive features (aligned as one) -> f32
__device__ __forceinline__ void kv8_ld4(const bf16_t* p, float (&x)[4]) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    x[0] = __uint_as_float(w.x << 16); x[1] = __uint_as_float(w.x & 0xffff0000u); x[2] = __uint_as_float(w.y << 16); x[3] = __uint_as_float(w.y & 0xffff0000u);
}
__device__ __forceinline__ void kv8_ld4(const float* p, float (&x)[4]) {
    const f32x4 w = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = w[e];
}
// 8 consecutive features (16-byte aligned) -> f32
template <typename T> __device__ __forceinline__ void kv8_ld8(const T* p, float (&x)[8]) { ld8(p, x); }
__device__ __forceinline__ void kv8_st16(void* p, size_t i, int bf16, const float (&x)[16]) {
    if (bf16) {
        u32x4* q = reinterpret_cast<u32x4*>(reinterpret_cast<bf16_t*>(p) + i);
#pragma unroll
        for (int h = 0; h < 2; ++h)
            q[h] = u32x4{pack_bf16x2(x[h * 8], x[h * 8 + 1]), pack_bf16x2(x[h * 8 + 2], x[h * 8 + 3]), pack_bf16x2(x[h * 8 + 4], x[h * 8 + 5]),
                         pack_bf16x2(x[h * 8 + 6], x[h * 8 + 7])};
    } else {
        f32x4* q = reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p) + i);
#pragma unroll
        for (int h = 0; h < 4; ++h) q[h] = f32x4{x[h * 4], x[h * 4 + 1], x[h * 4 + 2], x[h * 4 + 3]};
    }
}

// =====================================================================================================
// quantising a block
// =====================================================================================================
// The first 256 threads of a workgroup: a thread takes chunks of 16 features of a token, so loads and key codes are 16 bytes
// wide; the value codes are turned feature-major through LDS, 4 tokens x 4 features (words) at a time.
struct Kv8Scale { float scale, inv; };
__device__ __forceinline__ Kv8Scale kv8_scale(float amax) {   // +infinity: a NaN or an infinity among the values
    Kv8Scale s;
    if (amax == INFINITY) { s.scale = __uint_as_float(0x7fc00000u); s.inv = 0.f; }
    else if (amax < 7.52316384526264e-37f) { s.scale = 0.f; s.inv = 0.f; }   // 2^-120: 127 / amax stays finite above
    else { s.scale = __fdiv_rn(amax, 127.f); s.inv = __fdiv_rn(127.f, amax); }
    return s;
}
__device__ __forceinline__ float kv8_amax(float m, float v) {   // fmaxf would drop a NaN
    const float a = fabsf(v);
    return fmaxf(m, a <= 3.4028234663852886e38f ? a : INFINITY);
}
// 4 codes: the product rounded to f32, then to the nearest integer by adding 1.5 * 2^23 (ties to even; |product| <= 127 (1 + 2^-23)),
// whose low byte it then is
__device__ __forceinline__ uint32_t kv8_codes4(const float* x, float inv) {
    uint32_t b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = __float_as_uint(x[e] * inv + 12582912.f);
    return __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u) | __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
}
// 4 x 4 bytes: out word j = byte j of the four words
__device__ __forceinline__ void kv8_transpose4(const uint32_t (&w)[4], uint32_t (&o)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
    o[0] = __builtin_amdgcn_perm(b, a, 0x05040100u); o[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    o[2] = __builtin_amdgcn_perm(d, c, 0x05040100u); o[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

template <int HD> struct Kv8QuantLds { uint32_t v[BLK * (HD / 4 + 1)]; float red[2][4]; };

// load(part, token, feature, x): 16 features as the tail holds them.  Every thread of the workgroup has to come here.
template <int HD, typename G>
__device__ __forceinline__ void kv8_quantise_block(const acmi_kv8_cache& c, size_t hb, Kv8QuantLds<HD>& sm, const G& load) {
    constexpr int NCH = HD * BLK / 16, RND = NCH > 256 ? NCH / 256 : 1, PW = HD / 4 + 1;
    float x[2][RND][16], amax[2] = {0.f, 0.f};
    const int tid = threadIdx.x;
#pragma unroll
    for (int part = 0; part < 2; ++part)
#pragma unroll
        for (int q = 0; q < RND; ++q) {
            const int ch = q * 256 + tid;
            if (tid < 256 && ch < NCH) load(part, ch / (HD / 16), ch % (HD / 16) * 16, x[part][q]);
        }
#pragma unroll
    for (int part = 0; part < 2; ++part) {
#pragma unroll
        for (int q = 0; q < RND; ++q)
            if (tid < 256 && q * 256 + tid < NCH) {
#pragma unroll
                for (int j = 0; j < 16; ++j) amax[part] = kv8_amax(amax[part], x[part][q][j]);
            }
        amax[part] = wave_max(amax[part]);
        if ((tid & 63) == 0 && tid < 256) sm.red[part][tid >> 6] = amax[part];
    }
    __syncthreads();
    Kv8Scale s[2];
#pragma unroll
    for (int part = 0; part < 2; ++part) s[part] = kv8_scale(fmaxf(fmaxf(sm.red[part][0], sm.red[part][1]), fmaxf(sm.red[part][2], sm.red[part][3])));
    if (tid == 0) { c.k_scale[hb] = s[0].scale; c.v_scale[hb] = s[1].scale; }
    u32x4* kd = reinterpret_cast<u32x4*>(reinterpret_cast<uint8_t*>(c.k_codes) + hb * (size_t)(BLK * HD));
    uint32_t* vd = reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(c.v_codes) + hb * (size_t)(BLK * HD));
#pragma unroll
    for (int q = 0; q < RND; ++q) {
        const int ch = q * 256 + tid;
        if (tid < 256 && ch < NCH) {
            kd[ch] = u32x4{kv8_codes4(x[0][q], s[0].inv), kv8_codes4(x[0][q] + 4, s[0].inv), kv8_codes4(x[0][q] + 8, s[0].inv), kv8_codes4(x[0][q] + 12, s[0].inv)};
            uint32_t* l = sm.v + ch / (HD / 16) * PW + ch % (HD / 16) * 4;
#pragma unroll
            for (int k = 0; k < 4; ++k) l[k] = kv8_codes4(x[1][q] + 4 * k, s[1].inv);
        }
    }
    __syncthreads();
    if (tid < 256)
        for (int e = tid; e < HD / 4 * 16; e += 256) {   // (4 features f4, word w of their 64 bytes: tokens (w & 3) * 16 + (w >> 2) * 4 ..)
            const int w = e & 15, f4 = e >> 4, t = (w & 3) * 16 + (w >> 2) * 4;
            const uint32_t in[4] = {sm.v[t * PW + f4], sm.v[(t + 1) * PW + f4], sm.v[(t + 2) * PW + f4], sm.v[(t + 3) * PW + f4]};
            uint32_t o[4];
            kv8_transpose4(in, o);
#pragma unroll
            for (int j = 0; j < 4; ++j) vd[(f4 * 4 + j) * 16 + w] = o[j];
        }
}

// =====================================================================================================
// store
// =====================================================================================================
// One workgroup per (row, head, block that the call completes); workgroup 0 of a (row, head) also owns the tail: it first
// quantises the block that the old tail begins (reading the tail), then overwrites the tail with the newest block's tokens.
struct Kv8StoreArgs {
    acmi_kv8_cache c;
    const void* k; const void* v; int bf16;
    long long k_row, k_tok, k_head, v_row, v_tok, v_head;
    int L; const int* start; const int* n;
};

template <int HD>
__global__ __launch_bounds__(256) void kv8_store_kernel(const Kv8StoreArgs p) {
    __shared__ Kv8QuantLds<HD> sm;
    const int j = blockIdx.x, h = blockIdx.y, row = blockIdx.z;
    const int cap = p.c.nblk * BLK, tb = p.c.tail_dtype == ACMI_BF16;
    const int start = p.start != nullptr ? p.start[row] : 0;
    const int n = min(p.n != nullptr ? p.n[row] : p.L, p.L);
    if (start < 0 || start >= cap || n <= 0) return;
    const int end = (int)min((long long)start + n, (long long)cap);
    const int b0 = start / BLK, b1 = end / BLK, blk = b0 + j, last = (end - 1) / BLK;
    const size_t rh = (size_t)row * p.c.H + h, tbase = rh * (BLK * HD);
    const size_t kb = (size_t)(row * p.k_row + h * p.k_head), vb = (size_t)(row * p.v_row + h * p.v_head);
    auto fresh = [&](int part, int pos, int d, float (&x)[16]) {   // a token of this call, as the tail will hold it
        kv8_ld16(part == 0 ? p.k : p.v, (part == 0 ? kb : vb) + (size_t)(pos - start) * (part == 0 ? p.k_tok : p.v_tok) + d, p.bf16, x);
        if (tb && !p.bf16) {
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = kv8_round(x[e], 1);
        }
    };
    if (blk < b1)
        kv8_quantise_block<HD>(p.c, rh * p.c.nblk + blk, sm, [&](int part, int t, int d, float (&x)[16]) {
            const int pos = blk * BLK + t;
            if (pos < start) kv8_ld16(part == 0 ? p.c.k_tail : p.c.v_tail, tbase + t * HD + d, tb, x);
            else fresh(part, pos, d, x);
        });
    if (j == 0) {
        __syncthreads();   // the old tail has been read
        const int first = max(start, last * BLK);
        for (int e = threadIdx.x; e < (end - first) * (HD / 16); e += 256) {
            const int pos = first + e / (HD / 16), d = e % (HD / 16) * 16;
            const size_t at = tbase + (size_t)(pos % BLK) * HD + d;
            float x[16];
            fresh(0, pos, d, x);
            kv8_st16(p.c.k_tail, at, tb, x);
            fresh(1, pos, d, x);
            kv8_st16(p.c.v_tail, at, tb, x);
        }
    }
}

// =====================================================================================================
// load
// =====================================================================================================
struct Kv8LoadArgs { acmi_kv8_cache c; const int* len; int T; void* k; void* v; int bf16; };

__device__ __forceinline__ void kv8_st4(void* p, size_t i, int bf16, const f32x4& v) {
    if (bf16) *reinterpret_cast<uint2*>(reinterpret_cast<bf16_t*>(p) + i) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    else *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p) + i) = v;
}
__device__ __forceinline__ f32x4 kv8_values4(uint32_t w, float scale) {
    return f32x4{(float)(int8_t)w * scale, (float)(int8_t)(w >> 8) * scale, (float)(int8_t)(w >> 16) * scale, (float)(int8_t)(w >> 24) * scale};
}

// one workgroup per (row, head, block): a thread takes 4 features of 4 tokens, so every store of a wave is whole rows; the value
// codes come through LDS (pitch 17 words: conflict free) and are turned 4 x 4
template <int HD>
__global__ __launch_bounds__(256) void kv8_load_kernel(const Kv8LoadArgs p) {
    __shared__ uint32_t sv[HD * 17];
    const int blk = blockIdx.x, h = blockIdx.y, row = blockIdx.z;
    const int tb = p.c.tail_dtype == ACMI_BF16;
    const int len = max(0, min(p.len[row], p.c.nblk * BLK)), last = max(len - 1, 0) / BLK;
    const size_t rh = (size_t)row * p.c.H + h, hb = rh * p.c.nblk + blk, ob = rh * p.T * HD;
    if (blk < last) {
        const float ks = p.c.k_scale[hb], vs = p.c.v_scale[hb];
        const uint32_t* kc = reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint8_t*>(p.c.k_codes) + hb * (size_t)(BLK * HD));
        const u32x4* vc = reinterpret_cast<const u32x4*>(reinterpret_cast<const uint8_t*>(p.c.v_codes) + hb * (size_t)(BLK * HD));
        for (int e = threadIdx.x; e < HD * 4; e += 256) {
            const u32x4 w = vc[e];
#pragma unroll
            for (int j = 0; j < 4; ++j) sv[(e >> 2) * 17 + (e & 3) * 4 + j] = w[j];
        }
        for (int e = threadIdx.x; e < BLK * HD / 4; e += 256) {
            const int pos = blk * BLK + e / (HD / 4);
            if (pos < p.T) kv8_st4(p.k, ob + (size_t)pos * HD + e % (HD / 4) * 4, p.bf16, kv8_values4(kc[e], ks));
        }
        __syncthreads();
        for (int e = threadIdx.x; e < HD / 4 * 16; e += 256) {
            const int f4 = e % (HD / 4), w = e / (HD / 4), t = (w & 3) * 16 + (w >> 2) * 4;
            const uint32_t in[4] = {sv[(f4 * 4) * 17 + w], sv[(f4 * 4 + 1) * 17 + w], sv[(f4 * 4 + 2) * 17 + w], sv[(f4 * 4 + 3) * 17 + w]};
            uint32_t o[4];
            kv8_transpose4(in, o);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int pos = blk * BLK + t + j;
                if (pos < p.T) kv8_st4(p.v, ob + (size_t)pos * HD + f4 * 4, p.bf16, kv8_values4(o[j], vs));
            }
        }
        return;
    }
    for (int e = threadIdx.x; e < BLK * HD / 4; e += 256) {   // the newest block, and what lies past it
        const int t = e / (HD / 4), d = e % (HD / 4) * 4, pos = blk * BLK + t;
        if (pos >= p.T) break;
        f32x4 k = {0.f, 0.f, 0.f, 0.f}, v = k;
        if (pos < len) {
            const size_t at = rh * (BLK * HD) + t * HD + d;
#pragma unroll
            for (int j = 0; j < 4; ++j) { k[j] = kv8_ld(p.c.k_tail, at + j, tb); v[j] = kv8_ld(p.c.v_tail, at + j, tb); }
        }
        kv8_st4(p.k, ob + (size_t)pos * HD + d, p.bf16, k);
        kv8_st4(p.v, ob + (size_t)pos * HD + d, p.bf16, v);
    }
}

// =====================================================================================================
// attention
// =====================================================================================================
// Query columns: the S queries of the G heads that share a cache head, column c = query * G + head, in tiles of 16 (one MFMA
// dimension), so a block's codes are fetched and converted once for all of them.  Per block of 64 tokens
//     S^T[t, c] = sum_d K[t, d] Q[c, d]   (A operand: K codes, B operand: queries)     O^T[d, c] += sum_t V[t, d] P[t, c]
// Lane (kg = lane / 16, n = lane % 16) of the scores holds tokens tt * 16 + kg * 4 + r (tt, r < 4) of column n, and those
// probabilities are already the B operand of the second product, whose A operand is the 16 value codes of the lane (the order
// the codes are stored in).  Codes become f16 exactly: byte u = code + 128 under 0x64 is the f16 number 1024 + u, minus 1152.
// Queries are f16 relative to a power of two near the row's largest feature; an f32 query is a pair of f16 (22 bits).
// Per score the vector ALU does a maximum, one multiply-add (scale, running maximum), one exp2 and half a conversion: the value
// block's scale sits in the exponent too, relative to the largest p * scale met, and the row sums come out of the matrix cores (a
// product with ones), from the very f16 numbers that multiply the values.
struct Kv8AttnArgs {
    acmi_kv8_cache c;
    const void* q; int q_bf16; long long q_row, q_tok, q_head;
    int S, Hq, G;
    const int* len; int len_stride, len_bias; const int* q_len; const int* start_rows;
    int causal, past;
    const void* kn; const void* vn; int n_bf16; long long kn_row, kn_head, vn_row, vn_head;
    int complete;
    void* out; int out_mode, out_bf16, out_rbs, out_col0;
    float rG;   // 1 / G
    float* work; int splits, chunk, tiles;   // a row's blocks in chunks of `chunk`, one workgroup each
    float scale;
};

// 8 int8 codes -> 8 f16
__device__ __forceinline__ f16x8 kv8_cvt(uint32_t w0, uint32_t w1) {
    w0 ^= 0x80808080u; w1 ^= 0x80808080u;
    const f16x2 off = {(_Float16)1152.f, (_Float16)1152.f};
    const f16x2 a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w0, 0x04010400u)) - off;
    const f16x2 b = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w0, 0x04030402u)) - off;
    const f16x2 c = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w1, 0x04010400u)) - off;
    const f16x2 d = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w1, 0x04030402u)) - off;
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ f16x2 kv8_pk(float a, float b) { return __builtin_convertvector(kv8_f32x2{a, b}, f16x2); }   // nearest even
__device__ __forceinline__ f32x4 kv8_mma(const f16x8& a, const f16x8& b, const f32x4& c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

template <int HD> struct Kv8Geo {
    static constexpr int KW = HD >= 64 ? HD / 16 : 2;     // 32-bit words of K codes per lane and 16 tokens
    static constexpr int NK = KW / 2;                     // products of 32 features
    static constexpr int ND = HD / 16;                    // 16-feature tiles of O^T
};
// first of the 8 features that a lane's B operand of product k stands for (hd 16: lanes kg >= 2 hold nothing)
template <int HD> __device__ __forceinline__ int kv8_qdim(int kg, int k) {
    return HD >= 64 ? (k >> 1) * 64 + kg * 16 + (k & 1) * 8 : kg * 8;
}
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
// K codes of 16 tokens (lane: token nl), V codes of 16 features (lane: feature nl).  NT: as a stream -- not for the keys of hd 128,
// whose 128-byte rows take two requests: the line was gone before the second (decode over 32768 tokens: 70 -> 56 us)
template <int HD, bool NT>
__device__ __forceinline__ void kv8_fetch_k(const uint8_t* kb, int tt, int nl, int kg, uint32_t (&w)[Kv8Geo<HD>::KW]) {
    const uint8_t* row = kb + (tt * 16 + nl) * HD;
    if constexpr (HD >= 64) {
#pragma unroll
        for (int l = 0; l < HD / 64; ++l) {
            const u32x4* q = reinterpret_cast<const u32x4*>(row + l * 64 + kg * 16);
            const u32x4 v = NT ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[l * 4 + e] = v[e];
        }
    } else {   // hd 16: the queries of lanes kg >= 2 are 0, any code will do
        const u32x2* q = reinterpret_cast<const u32x2*>(row + (HD == 32 ? kg : (kg & 1)) * 8);
        const u32x2 v = NT ? __builtin_nontemporal_load(q) : *q;
        w[0] = v[0]; w[1] = v[1];
    }
}
template <bool NT>
__device__ __forceinline__ u32x4 kv8_fetch_v(const uint8_t* vb, int i, int nl, int kg) {
    const u32x4* q = reinterpret_cast<const u32x4*>(vb + (i * 16 + nl) * BLK + kg * 16);
    return NT ? __builtin_nontemporal_load(q) : *q;
}

// Probabilities are carried as 2^8 p relative to a running maximum that lags: it moves only when a block's maximum passes it by
// more than 2^7, so p <= 2^15 stays in f16's range and the sums are rescaled in the first block and almost never after.  f16
// resolves them down to 2^-32 of the maximum.
constexpr float KV8_PSHIFT = 8.f, KV8_LAG = 7.f;
// The unit of o goes down as well, where a block's value scale lies more than 2^10 below it: relative to it the block's probabilities
// would sink among the f16 subnormals (at 2^-10 the largest is 2^-2, a step 2^-24).  A unit is set by a scale, which tokens that are
// not seen or have no weight may have made large, so it says little about what o holds; o is f32 and may grow to 2^110.
constexpr float KV8_SINK = -10.f;

// 2^w = up / down: a unit near the largest number, times what a lagging maximum adds (2^7), leaves f32, and so may the quotient of an o
// that holds next to nothing in such a unit
struct Kv8Unit { float up, down; };
__device__ __forceinline__ Kv8Unit kv8_unit(float w) {
    const bool large = w > 64.f;
    return Kv8Unit{__builtin_amdgcn_exp2f(large ? w - 32.f : w), large ? 0x1p-32f : 1.f};
}

// one column tile's state: lane (kg, n) belongs to column n
template <int HD, bool QHL> struct Kv8Col {
    f16x8 qh[Kv8Geo<HD>::NK], ql[QHL ? Kv8Geo<HD>::NK : 1];
    float sfac;          // score factor: softmax scale * log2(e) * the query's power of two
    int lo, lim;         // positions [lo, lim) are seen
    float m, l;          // running maximum (log2 units, lagging); sum of 2^8 p
    float w;             // log2 of o's unit: like m, but for p times the block's value scale, and counted from m
    f32x4 o[Kv8Geo<HD>::ND];   // sum of 2^8 p v / 2^w
};

// A block of 64 tokens into QB column tiles.  K(tt, k) / V(i, u): the fragments (LO: KL / VL their f16 remainders, for a tail in
// f32); ks, vs: the block's scales; t0 its first position; after_k(): called once the K fragments have been used.
template <int HD, bool QHL, bool PHL, bool LO, int QB, typename FK, typename FV, typename FKL, typename FVL, typename FA, typename FS>
__device__ __forceinline__ void kv8_block(Kv8Col<HD, QHL> (&c)[QB], const FK& K, const FV& V, const FKL& KL, const FVL& VL,
                                          float ks, float vs, int t0, const FA& after_k, const FS& fix_scores) {
    constexpr int NK = Kv8Geo<HD>::NK, ND = Kv8Geo<HD>::ND;
    const int kg = (threadIdx.x & 63) >> 4;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    f32x4 s[QB][4];
    constexpr bool PRE = QB > 1 && NK <= 2;   // fragments from LDS: all requested at once, so that one latency is waited for
    f16x8 pre[PRE ? 4 : 1][PRE ? NK : 1];
    if constexpr (PRE) {
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
            for (int k = 0; k < NK; ++k) pre[tt][k] = K(tt, k);
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            f16x8 kf;
            if constexpr (PRE) kf = pre[tt][k];
            else kf = K(tt, k);
#pragma unroll
            for (int g = 0; g < QB; ++g) {
                s[g][tt] = kv8_mma(kf, c[g].qh[k], k == 0 ? zero : s[g][tt]);
                if constexpr (QHL) s[g][tt] = kv8_mma(kf, c[g].ql[k], s[g][tt]);
            }
            if constexpr (LO) {
                const f16x8 kl = KL(tt, k);
#pragma unroll
                for (int g = 0; g < QB; ++g) s[g][tt] = kv8_mma(kl, c[g].qh[k], s[g][tt]);
            }
        }
    after_k();
    fix_scores(s);
    const bool vnan = !(vs == vs);
    const float lv = vs > 0.f ? __builtin_amdgcn_logf(vs) : -300.f;   // log2; codes that are all 0 (or poisoned: below) count for nothing
    bool moved = false;
    f16x8 ph[QB][2], pl[QB][PHL ? 2 : 1];
    float shrink[QB];
#pragma unroll
    for (int g = 0; g < QB; ++g) {
        const int hi = c[g].lim - t0 - kg * 4, lo = c[g].lo - t0 - kg * 4;   // token tt * 16 + r of this lane is seen when lo <= it < hi
        if (__any(c[g].lim < t0 + BLK)) {
#pragma unroll
            for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[g][tt][r] = tt * 16 + r < hi ? s[g][tt][r] : -INFINITY;
        }
        if (__any(c[g].lo > t0)) {
#pragma unroll
            for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[g][tt][r] = tt * 16 + r >= lo ? s[g][tt][r] : -INFINITY;
        }
        float cmax = -INFINITY;
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) cmax = fmaxf(cmax, fmaxf(fmaxf(s[g][tt][0], s[g][tt][1]), fmaxf(s[g][tt][2], s[g][tt][3])));
        cmax = kv8_xmax(cmax);
        const bool none = cmax == -INFINITY;
        // a column that sees nothing here keeps clear of the block's scales (which a NaN may have poisoned); a key scale of 0
        // belongs to scores that are all 0
        float f = ks * c[g].sfac;
        if (f == 0.f) f = ks == 0.f ? 1.f : 1.17549435e-38f;   // (a product too small for f32: scores that are 0 beside a masked -infinity)
        f = none ? 1.f : f;
        const float top = cmax * f;
        const float m_new = top > c[g].m + KV8_LAG ? top : c[g].m;
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = __builtin_amdgcn_exp2f(c[g].m - m_use);
        // the numbers that multiply the values: p 2^d, d = the block's value scale against what o is counted in, so that neither
        // large values with small p nor small ones with large p leave f16's range
        const float w_old = top > c[g].m + KV8_LAG ? c[g].w - (m_new - c[g].m) : c[g].w;
        const float here = top - m_use + lv;
        float w_new = here > w_old + KV8_LAG ? here : w_old;
        const bool sink = lv < w_old + KV8_SINK;
        if (__any(sink)) {
            float omax = 0.f;
#pragma unroll
            for (int i = 0; i < ND; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) omax = fmaxf(omax, fabsf(c[g].o[i][r]) < INFINITY ? fabsf(c[g].o[i][r]) : 0.f);
            omax = kv8_xmax(omax);
            const float room = omax > 0.f ? fminf(110.f - (float)ilogbf(omax), 120.f) : 120.f;
            if (sink) w_new = fmaxf(here, w_old - room);
        }
        const float w_use = w_new == -INFINITY ? lv : w_new;
        shrink[g] = w_old - w_use;
        moved |= w_new != w_old;
        c[g].m = m_new;
        c[g].w = w_new;
        const float d = fmaxf(lv - w_use, -100.f);
        const float ie = __builtin_amdgcn_exp2f(-d);
        float base = d + KV8_PSHIFT - m_use, f2 = f;
        if (__any(fabsf(m_use) > 1024.f)) {
            // large scores: the multiply-add below subtracts the ROUNDED maximum from the exact product (and the shift drowns in it);
            // scaled and shifted apart, the largest score gives exactly 0
#pragma unroll
            for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[g][tt][r] = s[g][tt][r] * f - m_use;
            f2 = 1.f;
            base = d + KV8_PSHIFT;
        }
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[g][tt][r] = __builtin_amdgcn_exp2f(fmaf(s[g][tt][r], f2, base));
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float a = s[g][2 * u + (e >> 1)][(e & 1) * 2], b = s[g][2 * u + (e >> 1)][(e & 1) * 2 + 1];
                const f16x2 h = kv8_pk(a, b);
                ph[g][u][2 * e] = h[0]; ph[g][u][2 * e + 1] = h[1];
                if constexpr (PHL) {
                    const f16x2 w = kv8_pk(a - (float)h[0], b - (float)h[1]);
                    pl[g][u][2 * e] = w[0]; pl[g][u][2 * e + 1] = w[1];
                }
            }
        // the row sums: every row of (ones) P is the sum over the block's tokens
        float sum;
        if (!__any(d < KV8_SINK)) {   // (further down than o goes: nothing beside what it holds, but still itself in the sum l)
            const _Float16 o1 = (_Float16)1.f;
            const f16x8 ones = {o1, o1, o1, o1, o1, o1, o1, o1};
            f32x4 t = kv8_mma(ones, ph[g][1], kv8_mma(ones, ph[g][0], zero));
            if constexpr (PHL) t = kv8_mma(ones, pl[g][1], kv8_mma(ones, pl[g][0], t));
            sum = t[0];
        } else {
            sum = 0.f;
#pragma unroll
            for (int tt = 0; tt < 4; ++tt) sum += (s[g][tt][0] + s[g][tt][1]) + (s[g][tt][2] + s[g][tt][3]);
            sum += __shfl_xor(sum, 16, 64);
            sum += __shfl_xor(sum, 32, 64);
        }
        c[g].l = fmaf(c[g].l, alpha, sum * ie);
        if (vnan && !none) c[g].l = __uint_as_float(0x7fc00000u);
    }
    if (__any(moved)) {
#pragma unroll
        for (int g = 0; g < QB; ++g) {
            // in two steps where one factor would leave f32 (o itself, near 2^15, does not: it may have to come back)
            const bool far = shrink[g] < -100.f;
            const float f0 = __builtin_amdgcn_exp2f(far ? 0.5f * shrink[g] : shrink[g]), f1 = far ? f0 : 1.f;
#pragma unroll
            for (int i = 0; i < ND; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) c[g].o[i][r] = c[g].o[i][r] * f0 * f1;
        }
    }
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const f16x8 vf = V(i, u);
#pragma unroll
            for (int g = 0; g < QB; ++g) {
                c[g].o[i] = kv8_mma(vf, ph[g][u], c[g].o[i]);
                if constexpr (PHL) c[g].o[i] = kv8_mma(vf, pl[g][u], c[g].o[i]);
            }
            if constexpr (LO) {
                const f16x8 vl = VL(i, u);
#pragma unroll
                for (int g = 0; g < QB; ++g) c[g].o[i] = kv8_mma(vl, ph[g][u], c[g].o[i]);
            }
        }
}

// what a column is: row geometry shared by both kernels
// column -> query: exact for columns below 2^21 (checked by the entry), since (c + 1/2) / G is at least 1 / (2 G) from an integer
__device__ __forceinline__ int kv8_query(const Kv8AttnArgs& p, int c) { return (int)(((float)c + 0.5f) * p.rG); }

struct Kv8RowInfo { int len, qlen, start; bool fresh; };   // fresh: the call brings the row's newest token (and it fits)
__device__ __forceinline__ Kv8RowInfo kv8_row_of(const Kv8AttnArgs& p, int row, int len0) {
    Kv8RowInfo r;
    // (every load at once, then into scalar registers: what follows from them is the same for the whole wave)
    const int ql = p.q_len != nullptr ? p.q_len[row] : p.S;
    const int st = p.start_rows != nullptr ? p.start_rows[row] : 0;
    const long long len = (long long)__builtin_amdgcn_readfirstlane(len0) + p.len_bias;
    r.len = (int)max(0LL, min(len, (long long)p.c.nblk * BLK));
    r.fresh = p.kn != nullptr && r.len == len && len > 0;
    r.qlen = max(0, min(__builtin_amdgcn_readfirstlane(ql), p.S));
    r.start = max(0, __builtin_amdgcn_readfirstlane(st));
    return r;
}
__device__ __forceinline__ Kv8RowInfo kv8_row(const Kv8AttnArgs& p, int row) { return kv8_row_of(p, row, p.len[(size_t)row * p.len_stride]); }

// 8 NK query features of a lane at q + at: x[k][j] = feature kv8_qdim(kg, k) + j
template <int HD>
__device__ __forceinline__ void kv8_load_q(const void* q, size_t qb, int bf16, int kg, float (&x)[Kv8Geo<HD>::NK][8]) {
    u32x4 w[Kv8Geo<HD>::NK][2];
    if (bf16) {   // (requests only: a conversion here would wait for them)
#pragma unroll
        for (int k = 0; k < Kv8Geo<HD>::NK; ++k)
            w[k][0] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const bf16_t*>(q) + qb + (HD == 16 ? (kg & 1) * 8 : kv8_qdim<HD>(kg, k)));
    } else {
#pragma unroll
        for (int k = 0; k < Kv8Geo<HD>::NK; ++k) {
            const u32x4* s = reinterpret_cast<const u32x4*>(reinterpret_cast<const float*>(q) + qb + (HD == 16 ? (kg & 1) * 8 : kv8_qdim<HD>(kg, k)));
            w[k][0] = s[0]; w[k][1] = s[1];
        }
    }
#pragma unroll
    for (int k = 0; k < Kv8Geo<HD>::NK; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (bf16) { x[k][2 * e] = __uint_as_float(w[k][0][e] << 16); x[k][2 * e + 1] = __uint_as_float(w[k][0][e] & 0xffff0000u); }
            else { x[k][e] = __uint_as_float(w[k][0][e]); x[k][4 + e] = __uint_as_float(w[k][1][e]); }
        }
    if (HD == 16 && kg >= 2) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[0][j] = 0.f;
    }
}
// where column cidx's query lies (past the last column: some query)
__device__ __forceinline__ size_t kv8_query_at(const Kv8AttnArgs& p, int row, int kvh, int cidx) {
    const int s0 = kv8_query(p, cidx), g = cidx - s0 * p.G, s = min(s0, p.S - 1);
    return (size_t)(row * p.q_row + (long long)s * p.q_tok + (long long)(kvh * p.G + g) * p.q_head);
}

// column cidx of (row, cache head): visible range and operands from its features
template <int HD, bool QHL>
__device__ __forceinline__ void kv8_column(const Kv8AttnArgs& p, const Kv8RowInfo& ri, int cidx, const float (&x)[Kv8Geo<HD>::NK][8], Kv8Col<HD, QHL>& c) {
    const int s = kv8_query(p, cidx);
    const bool live = s < ri.qlen;
    const int pos = ri.len - ri.qlen + s;
    // (columns without a query are never stored: they see everything, so that they do not keep a block on the masked path)
    c.lim = !live ? 0x7fffffff : p.causal ? max(0, min(pos + 1, ri.len)) : ri.len;
    c.lo = live ? ri.start : 0;
    if (live && p.causal && p.past > 0) c.lo = max(c.lo, pos - p.past);
    if (c.lo >= c.lim) { c.lo = 0; c.lim = 0; }
    c.m = c.w = -INFINITY; c.l = 0.f;
#pragma unroll
    for (int i = 0; i < Kv8Geo<HD>::ND; ++i) c.o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float amax = 0.f, bad = 0.f;   // bad: NaN as soon as a feature is not finite (which a maximum would not tell)
#pragma unroll
    for (int k = 0; k < Kv8Geo<HD>::NK; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) { amax = fmaxf(amax, fabsf(x[k][j])); bad = fmaf(x[k][j], 0.f, bad); }
    amax = kv8_xmax(bad == 0.f ? amax : INFINITY);
    // features times a power of two that brings the largest into [2^14, 2^15); a query with a NaN or an infinity gives NaN
    const int e = (amax > 0.f && amax < INFINITY) ? ilogbf(amax) : 0;
    const float down = ldexpf(1.f, min(14 - e, 127));
    c.sfac = amax == INFINITY ? __uint_as_float(0x7fc00000u) : p.scale * 1.4426950408889634f / down;
#pragma unroll
    for (int k = 0; k < Kv8Geo<HD>::NK; ++k)
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const float y0 = amax == INFINITY ? 0.f : x[k][j] * down, y1 = amax == INFINITY ? 0.f : x[k][j + 1] * down;
            const f16x2 h = kv8_pk(y0, y1);
            c.qh[k][j] = h[0]; c.qh[k][j + 1] = h[1];
            if constexpr (QHL) {
                const f16x2 l = kv8_pk(y0 - (float)h[0], y1 - (float)h[1]);
                c.ql[k][j] = l[0]; c.ql[k][j + 1] = l[1];
            }
        }
}

// the blocks of codes a column tile visits, and how many workgroups share them
struct Kv8Span { int bf, bt, eff; bool live, tail; };
constexpr int KV8_MAX_SPLITS = 64;
// Workgroups that a split call aims at: two per CU, what its registers let run at once.  4 rows x 8 cache heads of 128 features, up
// to 32768 tokens, with the join: 512 40.8 us (256 40.3, within the noise, but half as many on a call whose rows differ in length),
// 1024 45.8.
constexpr int KV8_TARGET = 512;
__device__ __forceinline__ Kv8Span kv8_span(const Kv8AttnArgs& p, const Kv8RowInfo& ri, int c0, int c1) {   // columns [c0, c1)
    Kv8Span s;
    const int s0 = c0 / p.G, s1 = min((c1 - 1) / p.G, ri.qlen - 1);
    s.live = s0 <= s1 && ri.len > 0;
    s.bf = s.bt = 0; s.eff = 1; s.tail = false;
    if (!s.live) return s;
    const int nf = (ri.len - 1) / BLK, p0 = ri.len - ri.qlen + s0, p1 = ri.len - ri.qlen + s1;
    const int lim = p.causal ? max(0, p1 + 1) : ri.len;
    const int lo = max(ri.start, (p.causal && p.past > 0) ? p0 - p.past : 0);
    s.bt = min(nf, (lim + BLK - 1) / BLK);
    s.bf = min(lo / BLK, s.bt);
    s.eff = p.splits == 1 ? 1 : max(1, min(p.splits, (s.bt - s.bf + p.chunk - 1) / p.chunk));
    s.tail = lim > nf * BLK && lo < ri.len;
    return s;
}

typedef __bf16 kv8_bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t kv8_pack_bf16(float lo, float hi) {   // nearest even, one instruction
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(kv8_f32x2{lo, hi}, kv8_bf16x2));
}

// out of a finished column: 4 consecutive features
__device__ __forceinline__ void kv8_put4(const Kv8AttnArgs& p, int row, int s, int head, int HD, int d, const f32x4& v) {
    const size_t at = (((size_t)row * p.S + s) * p.Hq + head) * HD + d;
    if (p.out_mode == ACMI_OUT_F32) *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p.out) + at) = v;
    else if (p.out_mode == ACMI_OUT_BF16)
        *reinterpret_cast<uint2*>(reinterpret_cast<bf16_t*>(p.out) + at) = make_uint2(kv8_pack_bf16(v[0], v[1]), kv8_pack_bf16(v[2], v[3]));
    else {
        const int col = p.out_col0 + head * HD + d;   // (a multiple of 4: the four features share a lane's 16 bytes)
        if (p.out_bf16)
            *reinterpret_cast<uint2*>(reinterpret_cast<bf16_t*>(p.out) + tiled_index<bf16_t>(row, col, p.out_rbs)) =
                make_uint2(kv8_pack_bf16(v[0], v[1]), kv8_pack_bf16(v[2], v[3]));
        else *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p.out) + tiled_index<float>(row, col, p.out_rbs)) = v;
    }
}

// ---- few queries: one workgroup per (split, column tile of a cache head, row); its NW waves take the blocks in turn, the last four of
// them 16 tokens of the tail each, and are joined through LDS.  A wave keeps one block in flight: the next block's K is requested as
// soon as this block's K has been multiplied, its V likewise.  Bound by the codes' bytes: 4 rows of 9001 to 32768 tokens x 8 heads of
// 128, 171 MB in 35.6 us = 4.8 TB/s, the rate of a large copy; 64 rows of 750 x 24 heads of 64 3.9 TB/s; 16 rows of 750 2.3 TB/s.
// Launch bound per SIMD: a wave's block in flight takes 128 registers at 64 features, 226 at 128.  64 rows of 750 tokens x 24 heads of
// 64: 4 per SIMD 38 us, 2 41; up to 32768 tokens, hd 128, with the join: 2 per SIMD 40.8 us, 1 47.5.
template <int HD> constexpr int kv8_wpe() { return HD == 128 ? 2 : 4; }

__device__ __forceinline__ float raw8(bf16_t v) { return bf16_to_f32(v); }
__device__ __forceinline__ float raw8(float v) { return v; }

// 16 places of the tail as they are in memory: requested before anything else is known of the row (the places do not depend on
// its length), made into numbers when they are used.  Keys: lane (kg, nl) the features of its queries' lanes, of place nl;
// values: feature i * 16 + nl of places kg * 4 + r.
template <int HD> struct Kv8TailRaw { u32x4 k[Kv8Geo<HD>::NK][2]; uint32_t v[Kv8Geo<HD>::ND][4]; };
template <int HD>
__device__ __forceinline__ void kv8_tail_request(const void* kt, const void* vt, size_t base, int bf16, int nl, int kg, Kv8TailRaw<HD>& t) {
    constexpr int NK = Kv8Geo<HD>::NK, ND = Kv8Geo<HD>::ND;
    const size_t kb = base + (size_t)nl * HD, vb = base + (size_t)kg * 4 * HD + nl;
    if (bf16) {
#pragma unroll
        for (int k = 0; k < NK; ++k) t.k[k][0] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const bf16_t*>(kt) + kb + (HD == 16 ? (kg & 1) * 8 : kv8_qdim<HD>(kg, k)));
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < ND; ++i) t.v[i][r] = reinterpret_cast<const bf16_t*>(vt)[vb + r * HD + i * 16];
    } else {
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            const u32x4* q = reinterpret_cast<const u32x4*>(reinterpret_cast<const float*>(kt) + kb + (HD == 16 ? (kg & 1) * 8 : kv8_qdim<HD>(kg, k)));
            t.k[k][0] = q[0]; t.k[k][1] = q[1];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < ND; ++i) t.v[i][r] = reinterpret_cast<const uint32_t*>(vt)[vb + r * HD + i * 16];
    }
}

// The tail's 16 tokens slot0 .. in f32, through the f32 matrix instruction, before any block of codes.
template <int HD, bool QHL>
__device__ __forceinline__ void kv8_tail16(const Kv8AttnArgs& p, const Kv8RowInfo& ri, int row, int kvh, int slot0, const Kv8TailRaw<HD>& raw,
                                           const float (&x)[Kv8Geo<HD>::NK][8], Kv8Col<HD, QHL>& c) {
    constexpr int NK = Kv8Geo<HD>::NK, ND = Kv8Geo<HD>::ND;
    const int lane = threadIdx.x & 63, nl = lane & 15, kg = lane >> 4;
    const int last = (ri.len - 1) / BLK, t0 = last * BLK + slot0, tb = p.c.tail_dtype == ACMI_BF16;
    const size_t base = ((size_t)row * p.c.H + kvh) * (BLK * HD);
    const size_t kn0 = (size_t)(row * p.kn_row + kvh * p.kn_head), vn0 = (size_t)(row * p.vn_row + kvh * p.vn_head);
    float kx[NK][8], vx[ND][4];
    const int sh = tb ? 16 : 0;   // bf16 bits are the upper half of the f32
#pragma unroll
    for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (tb) { kx[k][2 * e] = __uint_as_float(raw.k[k][0][e] << 16); kx[k][2 * e + 1] = __uint_as_float(raw.k[k][0][e] & 0xffff0000u); }
            else { kx[k][e] = __uint_as_float(raw.k[k][0][e]); kx[k][4 + e] = __uint_as_float(raw.k[k][1][e]); }
        }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < ND; ++i) vx[i][r] = __uint_as_float(raw.v[i][r] << sh);
    // The row's newest token, which the tail does not hold yet, is put in its place.  (A token past the row's length: whatever the
    // tail holds there only reaches scores that are masked; its values are dropped.)
    if (ri.fresh && ri.len - 1 < t0 + 16) {   // (wave uniform; the newest token is never before t0)
        float kn[NK][8], vn[ND];
        auto from_new = [&](auto* k, auto* v) {
#pragma unroll
            for (int q = 0; q < NK; ++q) kv8_ld8(k + (HD == 16 ? (kg & 1) * 8 : kv8_qdim<HD>(kg, q)), kn[q]);
#pragma unroll
            for (int i = 0; i < ND; ++i) vn[i] = raw8(v[i * 16 + nl]);
        };
        if (p.n_bf16) from_new(reinterpret_cast<const bf16_t*>(p.kn) + kn0, reinterpret_cast<const bf16_t*>(p.vn) + vn0);
        else from_new(reinterpret_cast<const float*>(p.kn) + kn0, reinterpret_cast<const float*>(p.vn) + vn0);
        const int at = ri.len - 1 - t0;
#pragma unroll
        for (int k = 0; k < NK; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) kx[k][j] = nl == at ? kv8_round(kn[k][j], tb) : kx[k][j];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < ND; ++i) vx[i][r] = kg * 4 + r == at ? kv8_round(vn[i], tb) : vx[i][r];
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < ND; ++i) vx[i][r] = t0 + kg * 4 + r < ri.len ? vx[i][r] : 0.f;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) s = __builtin_amdgcn_mfma_f32_16x16x4f32(HD == 16 && kg >= 2 ? 0.f : kx[k][j], x[k][j], s, 0, 0, 0);
    const float f = p.scale * 1.4426950408889634f;
    float cmax = -INFINITY;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int t = t0 + kg * 4 + r;
        s[r] = (t >= c.lo && t < c.lim && t < ri.len) ? s[r] * f : -INFINITY;
        cmax = fmaxf(cmax, s[r]);
    }
    cmax = kv8_xmax(cmax);
    c.m = cmax;
    const float top = cmax == -INFINITY ? 0.f : cmax;
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) { s[r] = __builtin_amdgcn_exp2f(s[r] - top + KV8_PSHIFT); sum += s[r]; }
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    c.l = sum;
    float omax = 0.f;
    bool bad = false;   // a NaN or an infinity among the values: it must not meet the probability 0 of a column that does not see it
#pragma unroll
    for (int i = 0; i < ND; ++i) {
        f32x4 t = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float a = fabsf(vx[i][r]);
            const bool fin = a <= 3.4028234663852886e38f;
            bad |= !fin;
            t = __builtin_amdgcn_mfma_f32_16x16x4f32(fin ? vx[i][r] : 0.f, s[r] * 0x1p-12f, t, 0, 0, 0);   // p / 16: at most the largest value
        }
        c.o[i] = t;
#pragma unroll
        for (int r = 0; r < 4; ++r) omax = fmaxf(omax, fabsf(t[r]));
    }
    // o's unit is what the column holds, whatever there is that it does not see: a power of two that brings its largest feature to
    // [2^14, 2^15), where p = 1 of a block's largest code stands
    omax = kv8_xmax(omax);
    const int e = max(omax > 0.f ? ilogbf(omax) : -18, -118);
    c.w = c.m == -INFINITY ? -INFINITY : (float)(e - 2);
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) c.o[i][r] = ldexpf(c.o[i][r], 14 - e);
    if (__any(bad)) {   // those values one by one, each column for itself
        for (int tok = 0; tok < 16; ++tok) {
            float pr = 0.f;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float y = __shfl(s[r], (tok >> 2) * 16 + nl, 64);
                if ((tok & 3) == r) pr = y;
            }
            const int t = t0 + tok;
            const bool seen = t >= c.lo && t < c.lim && t < ri.len, isnew = ri.fresh && t == ri.len - 1;
#pragma unroll
            for (int i = 0; i < ND; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int d = i * 16 + kg * 4 + r;
                    float v = isnew ? kv8_round(kv8_ld(p.vn, vn0 + d, p.n_bf16), tb) : kv8_ld(p.c.v_tail, base + (size_t)(slot0 + tok) * HD + d, tb);
                    if (seen && !(fabsf(v) <= 3.4028234663852886e38f)) c.o[i][r] = fmaf(pr, v, c.o[i][r]);
                }
        }
    }
}

// Parts of a column are joined as they are, each in its unit: p v summed in absolute numbers would pass f32 where the quotient does not.
// dm: a part's maximum against the largest, w its unit, W the largest unit.
struct Kv8Joint { float l, o; };
__device__ __forceinline__ Kv8Joint kv8_joint(float dm, float w, float W) {
    return Kv8Joint{__builtin_amdgcn_exp2f(dm), __builtin_amdgcn_exp2f(dm + w - (W == -INFINITY ? 0.f : W))};
}

// The leading arguments are what the first requests need -- query, length word, tail -- and arrive in scalar registers at wave
// start (kernarg preload); the rest of the descriptor is fetched behind those requests.
//   g0 = H | G << 16   g1 = column tiles | q bf16 << 16 | tail bf16 << 17 | length per row << 18   query strides in elements
template <int HD, bool QHL, bool PHL, int NW>
__global__ __launch_bounds__(NW * 64, kv8_wpe<HD>()) void kv8_attn_split_kernel(const void* hq, const int* hlen, const void* hkt, const void* hvt,
                                                                                unsigned g0, unsigned g1, int q_row, int q_tok, int q_head, int S,
                                                                                const Kv8AttnArgs p) {
    constexpr int NK = Kv8Geo<HD>::NK, ND = Kv8Geo<HD>::ND, KW = Kv8Geo<HD>::KW, PITCH = HD + 4;
    __shared__ __attribute__((aligned(16))) float sm_o[NW][16][PITCH];
    __shared__ float sm_m[NW][16], sm_l[NW][16], sm_w[NW][16];
    __shared__ Kv8QuantLds<HD> sm_q;
    // (chunk slowest: the workgroups that a shorter row does not need come last, and leave at once)
    const int split = blockIdx.z, row = blockIdx.y;
    const int H = (int)(g0 & 0xffffu), G = (int)(g0 >> 16), qtiles = (int)(g1 & 0xffffu);
    const int kvh = blockIdx.x / qtiles, qt = blockIdx.x - kvh * qtiles;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nl = lane & 15, kg = lane >> 4;
    const int len0 = hlen[(g1 >> 18 & 1) ? row : 0];
    float x[NK][8];
    Kv8TailRaw<HD> raw;
    const bool early = g1 >> 19 & 1;
    const int tw = wave - (NW - 4);   // the last four waves take 16 places of the tail each (they have the fewer blocks)
    {
        // column -> query and head (a column past the last one reads some query of the call)
        const int cidx = qt * 16 + nl, sq = (int)(((float)cidx + 0.5f) * __builtin_amdgcn_rcpf((float)G)), g = cidx - sq * G;
        const size_t qb = (size_t)((long long)row * q_row + (long long)min(sq, S - 1) * q_tok + (long long)(kvh * G + g) * q_head);
        if (early && tw >= 0) kv8_tail_request<HD>(hkt, hvt, (((size_t)row * H + kvh) * BLK + tw * 16) * HD, g1 >> 17 & 1, nl, kg, raw);
        kv8_load_q<HD>(hq, qb, g1 >> 16 & 1, kg, x);
    }
    const Kv8RowInfo ri = kv8_row_of(p, row, len0);
    const Kv8Span sp = kv8_span(p, ri, qt * 16, min(qt * 16 + 16, p.S * p.G));
    if (split >= sp.eff) return;
    const bool mine = split == sp.eff - 1;   // the split that owns the tail
    const bool tail = mine && sp.tail && tw >= 0 && (ri.len - 1) / BLK * BLK + tw * 16 < ri.len;
    if (!early && tail) kv8_tail_request<HD>(hkt, hvt, (((size_t)row * H + kvh) * BLK + tw * 16) * HD, g1 >> 17 & 1, nl, kg, raw);
    const int s0 = sp.bf + split * p.chunk, s1 = sp.eff == 1 ? sp.bt : min(sp.bt, s0 + p.chunk);
    const size_t rh = (size_t)row * p.c.H + kvh, hb = rh * p.c.nblk;
    const uint8_t* kc = reinterpret_cast<const uint8_t*>(p.c.k_codes) + hb * (size_t)(BLK * HD);
    const uint8_t* vc = reinterpret_cast<const uint8_t*>(p.c.v_codes) + hb * (size_t)(BLK * HD);
    int z = 0;   // an opaque lane offset of 0: the scales come as vector loads, in order with the codes (a scalar load shares its
    asm volatile("" : "+v"(z));   // counter with the LDS and would be waited for early)
    const float* ks = p.c.k_scale + hb + z; const float* vs = p.c.v_scale + hb + z;

    uint32_t kr[4][KW];
    u32x4 vr[ND];
    float ksn = 0.f, vsn = 0.f;
    auto get_k = [&](int b) {
        const uint8_t* kb = kc + (size_t)b * (BLK * HD);
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) kv8_fetch_k<HD, HD <= 64>(kb, tt, nl, kg, kr[tt]);
        ksn = __builtin_nontemporal_load(ks + b);
        __builtin_amdgcn_sched_barrier(0);   // (the scheduler sinks requests to their uses)
    };
    auto get_v = [&](int b) {
        const uint8_t* vb = vc + (size_t)b * (BLK * HD);
#pragma unroll
        for (int i = 0; i < ND; ++i) vr[i] = kv8_fetch_v<true>(vb, i, nl, kg);
        vsn = __builtin_nontemporal_load(vs + b);
        __builtin_amdgcn_sched_barrier(0);
    };
    int b = s0 + wave;
    if (b < s1) { get_k(b); get_v(b); }
    Kv8Col<HD, QHL> c[1];
    kv8_column<HD, QHL>(p, ri, qt * 16 + nl, x, c[0]);
    if (tail) kv8_tail16<HD, QHL>(p, ri, row, kvh, tw * 16, raw, x, c[0]);
    while (b < s1) {
        // the next requests are not conditional (a wave's last ones read its last block again, from the cache): the waits of a
        // straight line count them exactly, those behind a branch would wait for everything
        const int nb = b + NW, rq = min(nb, s1 - 1);
        const float kcur = ksn, vcur = vsn;
        kv8_block<HD, QHL, PHL, false, 1>(c, [&](int tt, int k) { return kv8_cvt(kr[tt][2 * k], kr[tt][2 * k + 1]); },
                                          [&](int i, int u) { return kv8_cvt(vr[i][2 * u], vr[i][2 * u + 1]); }, 0, 0, kcur, vcur, b * BLK,
                                          [&] { get_k(rq); }, [](auto&) {});
        get_v(rq);
        b = nb;
    }
    // relative to the wave's maximum, in a unit near what the column holds (a scale may have set another: kv8_block)
    float omax = 0.f;
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) omax = fmaxf(omax, fabsf(c[0].o[i][r]));
    omax = kv8_xmax(omax);
    const int up = omax > 0.f && omax < INFINITY ? max(14 - ilogbf(omax), 0) : 0;
#pragma unroll
    for (int i = 0; i < ND; ++i) {
        f32x4 o = c[0].o[i];
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = ldexpf(o[r], up);
        *reinterpret_cast<f32x4*>(&sm_o[wave][nl][i * 16 + kg * 4]) = o;
    }
    if (kg == 0) { sm_m[wave][nl] = c[0].m; sm_l[wave][nl] = c[0].l; sm_w[wave][nl] = omax > 0.f ? c[0].w - (float)up : -INFINITY; }
    // the row's newest token and a block it completes (column tile 0 alone)
    if (mine && qt == 0 && ri.len > 0 && (ri.fresh || p.complete)) {
        const int tb = p.c.tail_dtype == ACMI_BF16;
        const size_t tbase = rh * (BLK * HD);
        auto newest = [&](int part, int d) {
            const long long i = (part == 0 ? row * p.kn_row + kvh * p.kn_head : row * p.vn_row + kvh * p.vn_head) + d;
            return kv8_ld(part == 0 ? p.kn : p.vn, (size_t)i, p.n_bf16);
        };
        if (ri.fresh && threadIdx.x < HD) {
            const size_t at = tbase + (size_t)((ri.len - 1) % BLK) * HD + threadIdx.x;
            kv8_st(p.c.k_tail, at, tb, newest(0, threadIdx.x));
            kv8_st(p.c.v_tail, at, tb, newest(1, threadIdx.x));
        }
        if (ri.len % BLK == 0)   // (workgroup uniform)
            kv8_quantise_block<HD>(p.c, hb + (ri.len - 1) / BLK, sm_q, [&](int part, int t, int d, float (&y)[16]) {
                if (t == BLK - 1 && ri.fresh) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) y[e] = kv8_round(newest(part, d + e), tb);
                } else {
                    kv8_ld16(part == 0 ? p.c.k_tail : p.c.v_tail, tbase + t * HD + d, tb, y);
                }
            });
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 16 * HD / 4; e += NW * 64) {
        const int n = e / (HD / 4), d = e % (HD / 4) * 4, cidx = qt * 16 + n;
        if (cidx >= p.S * p.G) continue;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, sm_m[w][n]);
        const float Mu = M == -INFINITY ? 0.f : M;
        float W = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) W = fmaxf(W, sm_m[w][n] - Mu + sm_w[w][n]);
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        float den = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const Kv8Joint j = kv8_joint(sm_m[w][n] - Mu, sm_w[w][n], W);
            const f32x4 y = *reinterpret_cast<const f32x4*>(&sm_o[w][n][d]);
            den = fmaf(j.l, sm_l[w][n], den);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = fmaf(j.o, y[r], o[r]);
        }
        if (sp.eff == 1) {
            const int s = kv8_query(p, cidx), g = cidx - s * p.G;
            const bool none = s >= ri.qlen || den == 0.f;
            const Kv8Unit unit = kv8_unit(W);
            den *= unit.down;
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = none ? 0.f : o[r] / den * unit.up;
            kv8_put4(p, row, s, kvh * p.G + g, HD, d, o);
        } else {   // partial: [row][cache head x tile][column][split][features | max, sum, unit]
            float* w = p.work + ((((size_t)row * gridDim.x + blockIdx.x) * 16 + n) * p.splits + split) * (HD + 4);
            *reinterpret_cast<f32x4*>(w + d) = o;
            if (d == 0) { w[HD] = M; w[HD + 1] = den; w[HD + 2] = W; }
        }
    }
}

// joins the splits of one column: 256 / (HD / 4) groups of threads take them in turn, then meet in LDS in a fixed order
template <int HD>
__global__ __launch_bounds__(256) void kv8_attn_join_kernel(const Kv8AttnArgs p) {
    constexpr int F4 = HD / 4, NG = 256 / F4;
    __shared__ __attribute__((aligned(16))) f32x4 so[NG][F4];
    __shared__ float sd[NG];
    const int n = blockIdx.x, row = blockIdx.z, qtiles = p.tiles, kvh = blockIdx.y / qtiles, qt = blockIdx.y - kvh * qtiles;
    const int cidx = qt * 16 + n;
    if (cidx >= p.S * p.G) return;
    const Kv8RowInfo ri = kv8_row(p, row);
    const Kv8Span sp = kv8_span(p, ri, qt * 16, min(qt * 16 + 16, p.S * p.G));
    if (sp.eff == 1) return;   // the split kernel has written it
    const float* w = p.work + (((size_t)row * gridDim.y + blockIdx.y) * 16 + n) * p.splits * (HD + 4);
    const int f4 = threadIdx.x % F4, grp = threadIdx.x / F4;
    const int lane = threadIdx.x & 63;
    const f32x4 mine = lane < sp.eff ? *reinterpret_cast<const f32x4*>(w + (size_t)lane * (HD + 4) + HD) : f32x4{-INFINITY, 0.f, -INFINITY, 0.f};   // (KV8_MAX_SPLITS = 64)
    const float M = wave_max(mine[0]), Mu = M == -INFINITY ? 0.f : M, W = wave_max(mine[0] - Mu + mine[2]);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float den = 0.f;
#pragma unroll 4
    for (int k = grp; k < sp.eff; k += NG) {
        const float* y = w + (size_t)k * (HD + 4);
        const Kv8Joint j = kv8_joint(y[HD] - Mu, y[HD + 2], W);
        const f32x4 v = *reinterpret_cast<const f32x4*>(y + f4 * 4);
        den = fmaf(j.l, y[HD + 1], den);
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = fmaf(j.o, v[r], o[r]);
    }
    so[grp][f4] = o;
    if (f4 == 0) sd[grp] = den;
    __syncthreads();
    if (grp != 0) return;
    for (int k = 1; k < NG; ++k) {
        den += sd[k];
        const f32x4 v = so[k][f4];
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] += v[r];
    }
    const int s = kv8_query(p, cidx), g = cidx - s * p.G;
    const bool none = s >= ri.qlen || den == 0.f;
    const Kv8Unit unit = kv8_unit(W);
    den *= unit.down;
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = none ? 0.f : o[r] / den * unit.up;
    kv8_put4(p, row, s, kvh * p.G + g, HD, f4 * 4, o);
}

// ---- many queries: a workgroup's 4 waves own QB column tiles each and walk the blocks together.  Every wave converts a quarter of
// the next block's codes to f16 fragments in LDS while this block is multiplied (two buffers, one barrier per block).  The tail
// is staged the same way, relative to a power of two, as f16 (bf16 tails: exact down to 2^-30 of the largest) or a pair of f16; where
// a token's features are all below 2^-12 of the tail's largest -- which this column may not see -- it takes kv8_tail_wide instead.
// Bound by vector issue beside the matrix cores: causal over 4096 tokens, 4 x 16 heads of 64, 605 TFLOP/s (f32 443).  Short calls
// are latencies one after another: 16 x 32 heads x 251 queries over 0 .. 77 states 20 us, of which the tail's staging is 6.
// All workgroups of a (row, cache head) run on one XCD (workgroup i on XCD i % 8), whose L2 then holds its codes; the last (causal:
// longest) tiles of all pairs go first, the short ones fill the end.
template <int HD> struct Kv8ManyLds {
    f16x8 k[2][4 * Kv8Geo<HD>::NK][64], v[2][2 * Kv8Geo<HD>::ND][64];
    float red[2][4];
    unsigned long long kbad, vbad;   // tokens of the tail that hold a NaN or an infinity
    int wide;                        // the tail's tokens differ too much in size for one unit
};

// The tail for one column tile in f32, 16 tokens at a time, straight from memory: a key or a value far larger than the rest
// must not cost the others their precision.  Values that are not finite are left out, as in the staged form.
template <int HD, bool QHL>
__device__ __forceinline__ void kv8_tail_wide(const Kv8AttnArgs& p, const Kv8RowInfo& ri, int row, int kvh, int cidx, Kv8Col<HD, QHL>& c) {
    constexpr int ND = Kv8Geo<HD>::ND;
    const int lane = threadIdx.x & 63, nl = lane & 15, kg = lane >> 4, tb = p.c.tail_dtype == ACMI_BF16;
    const int t0 = (ri.len - 1) / BLK * BLK;
    const size_t base = ((size_t)row * p.c.H + kvh) * (BLK * HD), qb = kv8_query_at(p, row, kvh, min(cidx, p.S * p.G - 1));
    const float f = c.sfac == c.sfac ? p.scale * 1.4426950408889634f : c.sfac;   // (NaN: a query that is not finite)
#pragma unroll 1
    for (int slot0 = 0; t0 + slot0 < ri.len; slot0 += 16) {
        f32x4 s = {0.f, 0.f, 0.f, 0.f}, t[ND];
#pragma unroll 1
        for (int d = 0; d < HD; d += 4)
            s = __builtin_amdgcn_mfma_f32_16x16x4f32(kv8_ld(p.c.k_tail, base + (size_t)(slot0 + nl) * HD + d + kg, tb), kv8_ld(p.q, qb + d + kg, p.q_bf16), s, 0, 0, 0);
        float cmax = -INFINITY, sum = 0.f, omax = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int at = t0 + slot0 + kg * 4 + r;
            s[r] = at >= c.lo && at < c.lim && at < ri.len ? s[r] * f : -INFINITY;
            cmax = fmaxf(cmax, s[r]);
        }
        cmax = kv8_xmax(cmax);
        const float m_new = fmaxf(cmax, c.m), m_use = m_new == -INFINITY ? 0.f : m_new;
        const float w_old = m_new > c.m ? c.w - (m_new - c.m) : c.w;
#pragma unroll
        for (int r = 0; r < 4; ++r) { s[r] = __builtin_amdgcn_exp2f(s[r] - m_use + KV8_PSHIFT); sum += s[r]; }
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        c.l = fmaf(c.l, __builtin_amdgcn_exp2f(c.m - m_use), sum);
        c.m = m_new;
#pragma unroll
        for (int i = 0; i < ND; ++i) {
            t[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int slot = slot0 + kg * 4 + r;
                const float v = t0 + slot < ri.len ? kv8_ld(p.c.v_tail, base + (size_t)slot * HD + i * 16 + nl, tb) : 0.f;
                t[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(fabsf(v) <= 3.4028234663852886e38f ? v : 0.f, s[r] * 0x1p-12f, t[i], 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) omax = fmaxf(omax, fabsf(t[i][r]));
        }
        omax = kv8_xmax(omax);
        // (o may stay in a unit far above what it holds: this is f32)
        const float w_new = fmaxf(w_old, omax > 0.f ? (float)(max(ilogbf(omax), -118) - 2) : m_new == -INFINITY ? -INFINITY : -120.f);
        const float sh = w_old == -INFINITY ? 0.f : w_old - w_new;
        const bool far = sh < -100.f;
        const float f0 = __builtin_amdgcn_exp2f(far ? 0.5f * sh : sh), f1 = far ? f0 : 1.f;
        const float up = w_new == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(-w_new);
#pragma unroll
        for (int i = 0; i < ND; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) c.o[i][r] = fmaf(t[i][r] * up, 4096.f, c.o[i][r] * f0 * f1);
        c.w = w_new;
    }
}

// Waves per SIMD: what the registers allow without spilling more than a few (hd 64, two tiles: 3 52.7 us, 2 61.9, for 600 tokens x
// 16 rows x 24 heads).
template <int HD, int QB> constexpr int kv8_many_wpe() { return HD == 128 ? 2 : QB == 2 ? 3 : 4; }
template <int HD, bool QHL, bool PHL, int QB>
__global__ __launch_bounds__(256, (kv8_many_wpe<HD, QB>())) void kv8_attn_many_kernel(const Kv8AttnArgs p) {
    constexpr int NK = Kv8Geo<HD>::NK, ND = Kv8Geo<HD>::ND, KW = Kv8Geo<HD>::KW, VT = ND >= 4 ? ND / 4 : 1;
    __shared__ Kv8ManyLds<HD> sm;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nl = lane & 15, kg = lane >> 4, cols = p.S * p.G;
    const int gpx = (p.c.rows * p.c.H + 7) >> 3, li = blockIdx.x >> 3, tq = li / gpx;   // (row, cache head) pairs per XCD
    const int grp = (blockIdx.x & 7) + 8 * (li - tq * gpx), tile = p.tiles - 1 - tq;
    if (grp >= p.c.rows * p.c.H) return;
    const int row = __builtin_amdgcn_readfirstlane(grp / p.c.H), kvh = grp - row * p.c.H;
    const int w0 = tile * 64 * QB, c0 = w0 + wave * 16 * QB;   // first column of the workgroup, of the wave
    const Kv8RowInfo ri = kv8_row(p, row);
    const Kv8Span sp = kv8_span(p, ri, w0, min(w0 + 64 * QB, cols));
    Kv8Span me = kv8_span(p, ri, min(c0, cols - 1), min(c0 + 16 * QB, cols));
    if (c0 >= cols) { me.live = me.tail = false; me.bf = me.bt = 0; }
    const size_t rh = (size_t)row * p.c.H + kvh, hb = rh * p.c.nblk;
    const uint8_t* kc = reinterpret_cast<const uint8_t*>(p.c.k_codes) + hb * (size_t)(BLK * HD);
    const uint8_t* vc = reinterpret_cast<const uint8_t*>(p.c.v_codes) + hb * (size_t)(BLK * HD);
    uint32_t kr[KW];
    u32x4 vr[VT];
    float ksn = 0.f, vsn = 0.f;
    int z = 0;   // an opaque lane offset of 0: vector loads, in order with the codes
    asm volatile("" : "+v"(z));
    auto request = [&](int b) {   // this wave's quarter: 16 tokens of K, VT feature tiles of V; the block's scales
        ksn = p.c.k_scale[hb + b + z];
        vsn = p.c.v_scale[hb + b + z];
        kv8_fetch_k<HD, false>(kc + (size_t)b * (BLK * HD), wave, nl, kg, kr);
#pragma unroll
        for (int q = 0; q < VT; ++q)
            if (wave + q * 4 < ND) vr[q] = kv8_fetch_v<false>(vc + (size_t)b * (BLK * HD), wave + q * 4, nl, kg);
    };
    auto stage = [&](int buf) {
#pragma unroll
        for (int k = 0; k < NK; ++k) sm.k[buf][wave * NK + k][lane] = kv8_cvt(kr[2 * k], kr[2 * k + 1]);
#pragma unroll
        for (int q = 0; q < VT; ++q)
            if (wave + q * 4 < ND) {
                sm.v[buf][(wave + q * 4) * 2][lane] = kv8_cvt(vr[q][0], vr[q][1]);
                sm.v[buf][(wave + q * 4) * 2 + 1][lane] = kv8_cvt(vr[q][2], vr[q][3]);
            }
    };
    auto none = [] {};
    auto keep = [](auto&) {};
    int buf = 0;
    float x[QB][NK][8];
#pragma unroll
    for (int g = 0; g < QB; ++g) kv8_load_q<HD>(p.q, kv8_query_at(p, row, kvh, c0 + g * 16 + nl), p.q_bf16, kg, x[g]);
    if (sp.bf < sp.bt) request(sp.bf);
    Kv8Col<HD, QHL> c[QB];
#pragma unroll
    for (int g = 0; g < QB; ++g) kv8_column<HD, QHL>(p, ri, c0 + g * 16 + nl, x[g], c[g]);
    if (sp.bf < sp.bt) {
        stage(0);
        __syncthreads();
        for (int b = sp.bf; b < sp.bt; ++b) {
            const bool more = b + 1 < sp.bt;
            const float ks = ksn, vs = vsn;
            if (more) request(b + 1);
            __builtin_amdgcn_sched_barrier(0);
            if (b >= me.bf && b < me.bt)
                kv8_block<HD, QHL, PHL, false, QB>(c, [&](int tt, int k) { return sm.k[buf][tt * NK + k][lane]; },
                                                   [&](int i, int u) { return sm.v[buf][i * 2 + u][lane]; }, 0, 0,
                                                   ks, vs, b * BLK, none, keep);
            if (more) stage(buf ^ 1);
            __syncthreads();
            buf ^= 1;
        }
    }
    if (sp.tail) {   // (workgroup uniform)
        const int tb = p.c.tail_dtype == ACMI_BF16, t0 = (ri.len - 1) / BLK * BLK, nt = ri.len - t0;
        const size_t base = rh * (BLK * HD);
        constexpr int UN = HD > 64 ? HD / 64 : 1;   // 4 tokens x 4 features of V per thread, so many times
        float kx[NK][8], vx[UN][4][4], ka = 0.f, va = 0.f;
        bool kb = false;
        unsigned long long vb = 0;
        if (threadIdx.x == 0) { sm.kbad = 0; sm.vbad = 0; sm.wide = 0; }
        const int tk = wave * 16 + nl;   // this lane's token of K
        auto from = [&](auto* kt, auto* vt) {   // every load of the tail in flight at once (places past the length are masked below)
#pragma unroll
            for (int k = 0; k < NK; ++k) kv8_ld8(kt + (size_t)tk * HD + (HD == 16 ? (kg & 1) * 8 : kv8_qdim<HD>(kg, k)), kx[k]);
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const int un = min(u * 256 + (int)threadIdx.x, HD * 4 - 1), t4 = un / (HD / 4) * 4, f4 = un % (HD / 4) * 4;
#pragma unroll
                for (int r = 0; r < 4; ++r) kv8_ld4(vt + (t4 + r) * HD + f4, vx[u][r]);
            }
        };
        if (tb) from(reinterpret_cast<const bf16_t*>(p.c.k_tail) + base, reinterpret_cast<const bf16_t*>(p.c.v_tail) + base);
        else from(reinterpret_cast<const float*>(p.c.k_tail) + base, reinterpret_cast<const float*>(p.c.v_tail) + base);
        float odd = 0.f;   // NaN as soon as a value is not finite
#pragma unroll
        for (int k = 0; k < NK; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                kx[k][j] = tk < nt ? kx[k][j] : 0.f;
                ka = fmaxf(ka, fabsf(kx[k][j]));
                odd = fmaf(kx[k][j], 0.f, odd);
            }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int t4 = min(u * 256 + (int)threadIdx.x, HD * 4 - 1) / (HD / 4) * 4;
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    vx[u][r][e] = t4 + r < nt ? vx[u][r][e] : 0.f;
                    va = fmaxf(va, fabsf(vx[u][r][e]));
                    odd = fmaf(vx[u][r][e], 0.f, odd);
                }
        }
        if (__any(odd != 0.f)) {   // those values are left out here, their tokens noted
            ka = va = 0.f;
#pragma unroll
            for (int k = 0; k < NK; ++k)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (!(fabsf(kx[k][j]) <= 3.4028234663852886e38f)) { kb = true; kx[k][j] = 0.f; }
                    ka = fmaxf(ka, fabsf(kx[k][j]));
                }
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const int t4 = min(u * 256 + (int)threadIdx.x, HD * 4 - 1) / (HD / 4) * 4;
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (!(fabsf(vx[u][r][e]) <= 3.4028234663852886e38f)) { vb |= 1ull << (t4 + r); vx[u][r][e] = 0.f; }
                        va = fmaxf(va, fabsf(vx[u][r][e]));
                    }
            }
        }
        const float kt = kv8_xmax(ka);   // of the token
        ka = wave_max(kt);
        va = wave_max(va);
        if (lane == 0) { sm.red[0][wave] = ka; sm.red[1][wave] = va; }
        __syncthreads();
        if (kb) atomicOr(&sm.kbad, 1ull << tk);
        if (vb != 0) atomicOr(&sm.vbad, vb);
        ka = fmaxf(fmaxf(sm.red[0][0], sm.red[0][1]), fmaxf(sm.red[0][2], sm.red[0][3]));
        va = fmaxf(fmaxf(sm.red[1][0], sm.red[1][1]), fmaxf(sm.red[1][2], sm.red[1][3]));
        bool wide = kt > 0.f && kt < ka * 0x1p-12f, few = false;
        float vt[UN][4];
#pragma unroll
        for (int u = 0; u < UN; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                vt[u][r] = fmaxf(fmaxf(fabsf(vx[u][r][0]), fabsf(vx[u][r][1])), fmaxf(fabsf(vx[u][r][2]), fabsf(vx[u][r][3])));
                few |= vt[u][r] > 0.f && vt[u][r] < va * 0x1p-12f;
            }
        if (__any(few)) {   // four features of a token: is it all of them (on the HD / 4 lanes next to each other)
#pragma unroll
            for (int u = 0; u < UN; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float t = vt[u][r];
#pragma unroll
                    for (int x = 1; x < HD / 4; x <<= 1) t = fmaxf(t, __shfl_xor(t, x, 64));
                    wide |= u * 256 + (int)threadIdx.x < HD * 4 && t > 0.f && t < va * 0x1p-12f;
                }
        }
        if (wide) sm.wide = 1;
        const float ku = ldexpf(1.f, min(14 - (ka > 0.f ? ilogbf(ka) : 0), 126)), vu = ldexpf(1.f, min(14 - (va > 0.f ? ilogbf(va) : 0), 126));
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            f16x8 h;
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                kx[k][j] *= ku; kx[k][j + 1] *= ku;
                const f16x2 y = kv8_pk(kx[k][j], kx[k][j + 1]);
                h[j] = y[0]; h[j + 1] = y[1];
            }
            sm.k[0][wave * NK + k][lane] = h;
            if (!tb) {
                f16x8 l;
#pragma unroll
                for (int j = 0; j < 8; ++j) l[j] = (_Float16)(kx[k][j] - (float)h[j]);
                sm.k[1][wave * NK + k][lane] = l;
            }
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int un = u * 256 + (int)threadIdx.x, t4 = un / (HD / 4), f = un % (HD / 4) * 4;
            if (un < HD * 4)
#pragma unroll
                for (int e = 0; e < 4; ++e) {   // feature f + e of tokens 4 t4 ..: half a lane's operand
                    const int at = (f >> 4) * 2 + (t4 >> 3), ln = (t4 & 3) * 16 + (f & 15) + e, half = (t4 >> 2) & 1;
                    f16x4 h;
#pragma unroll
                    for (int r = 0; r < 4; r += 2) {
                        vx[u][r][e] *= vu; vx[u][r + 1][e] *= vu;
                        const f16x2 y = kv8_pk(vx[u][r][e], vx[u][r + 1][e]);
                        h[r] = y[0]; h[r + 1] = y[1];
                    }
                    reinterpret_cast<f16x4*>(&sm.v[0][at][ln])[half] = h;
                    if (!tb) {
                        f16x4 l;
#pragma unroll
                        for (int r = 0; r < 4; ++r) l[r] = (_Float16)(vx[u][r][e] - (float)h[r]);
                        reinterpret_cast<f16x4*>(&sm.v[1][at][ln])[half] = l;
                    }
                }
        }
        __syncthreads();
        if (me.tail) {
            // tokens past the row's length are masked for every stored column by its limit; a column without a query may count them
            const unsigned long long kbad = sm.kbad, vbad = sm.vbad;
            const float ks = 1.f / ku, vs = 1.f / vu;
            // a score from the features themselves, for the tokens whose f16 fragments leave a value out
            auto dot = [&](int g, int t) {
                const int cidx = min(c0 + g * 16 + nl, cols - 1);
                const size_t qb = (size_t)(row * p.q_row + (long long)(cidx / p.G) * p.q_tok + (long long)(kvh * p.G + cidx % p.G) * p.q_head);
                float x = 0.f;
#pragma unroll 1
                for (int d = 0; d < HD; ++d) x = fmaf(kv8_ld(p.q, qb + d, p.q_bf16), kv8_ld(p.c.k_tail, base + (size_t)t * HD + d, tb), x);
                return x;
            };
            auto fix = [&](f32x4 (&s)[QB][4]) {
                if (kbad == 0) return;
#pragma unroll 1
                for (int t = 0; t < nt; ++t) {
                    if (!(kbad >> t & 1)) continue;
#pragma unroll
                    for (int g = 0; g < QB; ++g) {
                        const float x = dot(g, t);   // an infinity or a NaN, whatever its factor
#pragma unroll
                        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (tt * 16 + kg * 4 + r == t) s[g][tt][r] = x;
                    }
                }
            };
            auto K = [&](int tt, int k) { return sm.k[0][tt * NK + k][lane]; };
            auto V = [&](int i, int u) { return sm.v[0][i * 2 + u][lane]; };
            auto KL = [&](int tt, int k) { return sm.k[1][tt * NK + k][lane]; };
            auto VL = [&](int i, int u) { return sm.v[1][i * 2 + u][lane]; };
            if (sm.wide) {   // (workgroup uniform)
#pragma unroll
                for (int g = 0; g < QB; ++g) kv8_tail_wide<HD, QHL>(p, ri, row, kvh, c0 + g * 16 + nl, c[g]);
            } else if (tb) kv8_block<HD, QHL, PHL, false, QB>(c, K, V, 0, 0, ks, vs, t0, none, fix);
            else kv8_block<HD, QHL, PHL, true, QB>(c, K, V, KL, VL, ks, vs, t0, none, fix);
#pragma unroll 1
            for (int t = 0; t < (vbad != 0 ? nt : 0); ++t) {   // values that are not finite one by one, each column for itself
                if (!(vbad >> t & 1)) continue;
#pragma unroll
                for (int g = 0; g < QB; ++g) {
                    const float pr = __builtin_amdgcn_exp2f(dot(g, t) * (p.scale * 1.4426950408889634f) - c[g].m + KV8_PSHIFT);
                    const bool seen = t0 + t >= c[g].lo && t0 + t < c[g].lim;
#pragma unroll
                    for (int i = 0; i < ND; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float v = kv8_ld(p.c.v_tail, base + (size_t)t * HD + i * 16 + kg * 4 + r, tb);
                            if (seen && !(fabsf(v) <= 3.4028234663852886e38f)) c[g].o[i][r] = fmaf(pr, v, c[g].o[i][r]);
                        }
                }
            }
        }
    }
#pragma unroll
    for (int g = 0; g < QB; ++g) {
        const int cidx = c0 + g * 16 + nl, s = kv8_query(p, cidx), h = cidx - s * p.G;
        if (cidx >= cols) continue;
        const bool zero = s >= ri.qlen || c[g].l == 0.f;
        const Kv8Unit unit = kv8_unit(c[g].w);
        const float inv = 1.f / (c[g].l * unit.down);
#pragma unroll
        for (int i = 0; i < ND; ++i) {
            f32x4 o;
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = zero ? 0.f : c[g].o[i][r] * inv * unit.up;
            kv8_put4(p, row, s, kvh * p.G + h, HD, i * 16 + kg * 4, o);
        }
    }
}

// =====================================================================================================
// C entries
// =====================================================================================================
static int kv8_check(const acmi_kv8_cache* c, const char* who) {
    ACMI_REQUIRE(c != nullptr, "%s: null cache", who);
    ACMI_REQUIRE(c->hd == 16 || c->hd == 32 || c->hd == 64 || c->hd == 128, "%s: head dim %d unsupported (16, 32, 64, 128)", who, c->hd);
    ACMI_REQUIRE(c->rows > 0 && c->rows <= 65535 && c->H > 0 && c->H <= 65535 && c->nblk > 0 && c->nblk < (1 << 24),
                 "%s: bad cache shape rows=%d H=%d nblk=%d", who, c->rows, c->H, c->nblk);
    ACMI_REQUIRE(c->tail_dtype == ACMI_F32 || c->tail_dtype == ACMI_BF16, "%s: tail_dtype %d", who, c->tail_dtype);
    ACMI_REQUIRE(c->k_codes && c->v_codes && c->k_scale && c->v_scale && c->k_tail && c->v_tail, "%s: null cache buffer", who);
    ACMI_REQUIRE(((reinterpret_cast<size_t>(c->k_codes) | reinterpret_cast<size_t>(c->v_codes) | reinterpret_cast<size_t>(c->k_tail) |
                   reinterpret_cast<size_t>(c->v_tail)) & 15) == 0, "%s: codes and tails must be 16-byte aligned", who);
    return ACMI_OK;
}
static bool kv8_dtype_ok(int d) { return d == ACMI_F32 || d == ACMI_BF16; }
static bool kv8_rows_ok(const void* p, int es, long long a, long long b, long long c) {
    return ((reinterpret_cast<size_t>(p) | (size_t)(a * es) | (size_t)(b * es) | (size_t)(c * es)) & 15) == 0;
}

#define KV8_HD_SWITCH(hd, CASE) \
    switch (hd) {               \
        CASE(16)                \
        CASE(32)                \
        CASE(64)                \
        CASE(128)               \
        default: break;         \
    }

extern "C" int acmi_kv8_store(const acmi_kv8_cache* cache, const acmi_kv8_store_desc* desc, void* stream) {
    if (int rc = kv8_check(cache, "acmi_kv8_store")) return rc;
    ACMI_REQUIRE(desc != nullptr, "acmi_kv8_store: null descriptor");
    ACMI_REQUIRE(desc->L >= 0 && desc->L <= (1 << 30) && kv8_dtype_ok(desc->dtype), "acmi_kv8_store: L=%d dtype=%d", desc->L, desc->dtype);
    if (desc->L == 0) return ACMI_OK;
    ACMI_REQUIRE(desc->k && desc->v, "acmi_kv8_store: null k or v");
    const int es = desc->dtype == ACMI_BF16 ? 2 : 4;
    ACMI_REQUIRE(kv8_rows_ok(desc->k, es, desc->k_row, desc->k_tok, desc->k_head) && kv8_rows_ok(desc->v, es, desc->v_row, desc->v_tok, desc->v_head),
                 "acmi_kv8_store: k and v need 16-byte aligned rows");
    Kv8StoreArgs a = {};
    a.c = *cache; a.k = desc->k; a.v = desc->v; a.bf16 = desc->dtype == ACMI_BF16;
    a.k_row = desc->k_row; a.k_tok = desc->k_tok; a.k_head = desc->k_head;
    a.v_row = desc->v_row; a.v_tok = desc->v_tok; a.v_head = desc->v_head;
    a.L = desc->L; a.start = desc->start; a.n = desc->n;
    const int nb = min(desc->L / BLK + 2, cache->nblk);   // blocks a run of L tokens can touch
    const dim3 grid(nb, cache->H, cache->rows);
#define KV8_CASE(HDv) case HDv: hipLaunchKernelGGL((kv8_store_kernel<HDv>), grid, dim3(256), 0, (hipStream_t)stream, a); break;
    KV8_HD_SWITCH(cache->hd, KV8_CASE)
#undef KV8_CASE
    return acmi_check_launch("kv8_store_kernel");
}

extern "C" int acmi_kv8_load(const acmi_kv8_cache* cache, const int* len, int T, void* k_out, void* v_out, int out_dtype, void* stream) {
    if (int rc = kv8_check(cache, "acmi_kv8_load")) return rc;
    ACMI_REQUIRE(len != nullptr && T >= 0 && T <= cache->nblk * BLK && kv8_dtype_ok(out_dtype), "acmi_kv8_load: T=%d outside [0, %d] or dtype %d",
                 T, cache->nblk * BLK, out_dtype);
    if (T == 0) return ACMI_OK;
    ACMI_REQUIRE(k_out && v_out && ((reinterpret_cast<size_t>(k_out) | reinterpret_cast<size_t>(v_out)) & 15) == 0,
                 "acmi_kv8_load: outputs must be 16-byte aligned");
    Kv8LoadArgs a = {};
    a.c = *cache; a.len = len; a.T = T; a.k = k_out; a.v = v_out; a.bf16 = out_dtype == ACMI_BF16;
    const dim3 grid((T + BLK - 1) / BLK, cache->H, cache->rows);
#define KV8_CASE(HDv) case HDv: hipLaunchKernelGGL((kv8_load_kernel<HDv>), grid, dim3(256), 0, (hipStream_t)stream, a); break;
    KV8_HD_SWITCH(cache->hd, KV8_CASE)
#undef KV8_CASE
    return acmi_check_launch("kv8_load_kernel");
}

// The split form: one query per head (it alone stores a new token), one column tile, or few workgroups, three per CU -- a workgroup of
// it has a column tile and its waves share the blocks, where the prompt form's waves walk all blocks with a tile each.  Measured, us
// split / prompt form, in a graph: 4 x 8 heads x 128 queries of 300 (256 workgroups) 7.1 / 10.8, 1 x 16 x 600 of 600 (608) 11.1 /
// 15.5, 1 x 8 x 128 of 8000 (64) 19.1 / 116, 16 x 24 x 29 of 600 (768) 15.4 / 19.7; 8 x 8 x 200 of 600 (832) 16.1 / 16.0,
// 16 x 12 x 77 of 251 (960) 13.0 / 12.0, 64 x 8 x 4 x 16 of 1000 (2048) 52.1 / 28.5
constexpr int KV8_SPLIT_WGS = 768;
static bool kv8_few(const acmi_kv8_cache* c, int S, int G) {
    const long long tiles = ((long long)S * G + 15) / 16;
    return S == 1 || tiles == 1 || tiles * c->H * c->rows <= KV8_SPLIT_WGS;
}
// Blocks per workgroup: the longest possible row in so many chunks that the call has about KV8_TARGET workgroups; one chunk (and
// no second launch) when the tiles alone fill the chip.  The rows' lengths are not known here: shorter rows take fewer chunks of
// the same size, so that all workgroups take equally long.  A chunk is at least a block per wave, and a row of less than four per wave
// is not split: the second launch costs 4 us.  us in a graph, caches cold, unsplit / as here: 2 rows x 16 heads of 64 x 2800
// tokens 15.9 / 12.3, 7 x 2 x 3700 18.5 / 10.9, 4 x 8 x 4 heads of 128 x 2000 22.4 / 16.9; 2 x 16 x 1400 unsplit 11.1, split 12.7
static void kv8_split_plan(const acmi_kv8_cache* c, int S, int G, int* splits, int* chunk) {
    const long long tiles = (long long)c->H * ((S * G + 15) / 16) * c->rows;
    long long n = 1;
    const int least = c->hd == 128 ? 4 : 8;
    if (tiles * 4 <= KV8_TARGET && c->nblk >= 4 * least) n = max(1LL, min(min(KV8_TARGET / tiles, (long long)(c->nblk / least)), (long long)KV8_MAX_SPLITS));
    *chunk = (int)((c->nblk + n - 1) / n);
    *splits = (c->nblk + *chunk - 1) / *chunk;
}

extern "C" size_t acmi_kv8_attn_work_floats(const acmi_kv8_cache* cache, int S, int Hq) {
    if (kv8_check(cache, "acmi_kv8_attn_work_floats") || S <= 0 || Hq <= 0 || Hq % cache->H) return 0;
    const int G = Hq / cache->H;
    if (!kv8_few(cache, S, G)) return 0;
    int sp, chunk;
    kv8_split_plan(cache, S, G, &sp, &chunk);
    return sp == 1 ? 0 : (size_t)cache->rows * cache->H * ((S * G + 15) / 16) * sp * 16 * (cache->hd + 4);
}

extern "C" int acmi_kv8_attn(const acmi_kv8_cache* cache, const acmi_kv8_attn_desc* desc, void* stream) {
    if (int rc = kv8_check(cache, "acmi_kv8_attn")) return rc;
    ACMI_REQUIRE(desc != nullptr, "acmi_kv8_attn: null descriptor");
    const acmi_kv8_attn_desc& d = *desc;
    ACMI_REQUIRE(d.S >= 0 && d.S <= (1 << 20) && d.Hq > 0 && d.Hq % cache->H == 0 && d.Hq <= 65535, "acmi_kv8_attn: S=%d Hq=%d with %d cache heads", d.S, d.Hq, cache->H);
    if (d.S == 0) return ACMI_OK;
    ACMI_REQUIRE(d.q && d.out && d.len && (d.len_stride == 0 || d.len_stride == 1), "acmi_kv8_attn: null q, out or len, or len_stride %d", d.len_stride);
    ACMI_REQUIRE(kv8_dtype_ok(d.q_dtype), "acmi_kv8_attn: q_dtype %d", d.q_dtype);
    ACMI_REQUIRE(d.out_mode == ACMI_OUT_F32 || d.out_mode == ACMI_OUT_BF16 || (d.out_mode == ACMI_OUT_TILED && d.S == 1 && kv8_dtype_ok(d.out_dtype)),
                 "acmi_kv8_attn: out_mode %d out_dtype %d with S=%d", d.out_mode, d.out_dtype, d.S);
    ACMI_REQUIRE((reinterpret_cast<size_t>(d.out) & 15) == 0, "acmi_kv8_attn: out must be 16-byte aligned");
    ACMI_REQUIRE((d.k_new == nullptr) == (d.v_new == nullptr), "acmi_kv8_attn: k_new and v_new come together");
    ACMI_REQUIRE((d.k_new == nullptr && !d.complete) || (d.S == 1 && d.causal), "acmi_kv8_attn: a new token needs S = 1 and causal");
    ACMI_REQUIRE(d.k_new == nullptr || kv8_dtype_ok(d.new_dtype), "acmi_kv8_attn: new_dtype %d", d.new_dtype);
    ACMI_REQUIRE(kv8_rows_ok(d.q, d.q_dtype == ACMI_BF16 ? 2 : 4, d.q_row, d.S > 1 ? d.q_tok : 0, d.q_head), "acmi_kv8_attn: q needs 16-byte aligned rows");
    ACMI_REQUIRE(d.k_new == nullptr || (kv8_rows_ok(d.k_new, d.new_dtype == ACMI_BF16 ? 2 : 4, d.kn_row, d.kn_head, 0) &&
                                        kv8_rows_ok(d.v_new, d.new_dtype == ACMI_BF16 ? 2 : 4, d.vn_row, d.vn_head, 0)),
                 "acmi_kv8_attn: k_new and v_new need 16-byte aligned rows");
    ACMI_REQUIRE(d.past_context >= 0 && (d.past_context == 0 || d.causal), "acmi_kv8_attn: past_context=%d needs causal", d.past_context);
    Kv8AttnArgs a = {};
    a.c = *cache; a.q = d.q; a.q_bf16 = d.q_dtype == ACMI_BF16; a.q_row = d.q_row; a.q_tok = d.q_tok; a.q_head = d.q_head;
    a.S = d.S; a.Hq = d.Hq; a.G = d.Hq / cache->H; a.rG = 1.0f / (float)a.G;
    ACMI_REQUIRE((long long)d.S * a.G <= (1 << 21), "acmi_kv8_attn: S=%d x %d query heads per cache head (at most 2^21)", d.S, a.G);
    a.len = d.len; a.len_stride = d.len_stride; a.len_bias = d.len_bias; a.q_len = d.q_len; a.start_rows = d.start_rows;
    a.causal = d.causal != 0; a.past = d.past_context;
    a.kn = d.k_new; a.vn = d.v_new; a.n_bf16 = d.new_dtype == ACMI_BF16;
    a.kn_row = d.kn_row; a.kn_head = d.kn_head; a.vn_row = d.vn_row; a.vn_head = d.vn_head; a.complete = d.complete;
    a.out = d.out; a.out_mode = d.out_mode; a.out_bf16 = d.out_dtype == ACMI_BF16; a.out_col0 = d.out_col0;
    const int kt = d.out_dtype == ACMI_BF16 ? 32 : 16;
    a.out_rbs = d.out_rbs > 0 ? d.out_rbs : (d.Hq * cache->hd + kt - 1) / kt;
    if (d.out_mode == ACMI_OUT_TILED)
        ACMI_REQUIRE(d.out_col0 >= 0 && d.out_col0 % kt == 0 && (long long)a.out_rbs * kt >= (long long)d.out_col0 + d.Hq * cache->hd,
                     "acmi_kv8_attn: tiled output placement col0=%d rbs=%d does not hold %d columns", d.out_col0, a.out_rbs, d.Hq * cache->hd);
    a.scale = 1.0f / sqrtf((float)cache->hd);
    const bool out_f32 = d.out_mode == ACMI_OUT_F32 || (d.out_mode == ACMI_OUT_TILED && d.out_dtype == ACMI_F32);
    const bool qhl = d.q_dtype == ACMI_F32 || out_f32;   // (a bf16 query is one f16 exactly)
    hipStream_t st = (hipStream_t)stream;
    const int qtiles = (d.S * a.G + 15) / 16;
    const bool narrow = d.q_row == (int)d.q_row && (d.S == 1 || d.q_tok == (int)d.q_tok) && d.q_head == (int)d.q_head;   // query strides below 2^31
    if (kv8_few(cache, d.S, a.G) && (narrow || d.S == 1)) {
        kv8_split_plan(cache, d.S, a.G, &a.splits, &a.chunk);
        a.work = d.work;
        ACMI_REQUIRE(a.splits == 1 || (d.work != nullptr && (reinterpret_cast<size_t>(d.work) & 15) == 0),
                     "acmi_kv8_attn: needs acmi_kv8_attn_work_floats floats of 16-byte aligned work");
        ACMI_REQUIRE((long long)cache->H * qtiles <= 65535, "acmi_kv8_attn: %d heads x %d column tiles", cache->H, qtiles);
        const dim3 grid(cache->H * qtiles, cache->rows, a.splits);
        a.tiles = qtiles;
        ACMI_REQUIRE(narrow && a.G <= 65535, "acmi_kv8_attn: query strides beyond 2^31 elements, or %d query heads per cache head", a.G);
        const unsigned g0 = (unsigned)cache->H | (unsigned)a.G << 16;
        // A grid of at most one workgroup per CU is one chain of latencies: 8 waves share the blocks, and the tail is requested before
        // the row's length is known.  Larger grids are bytes: 4 waves, twice the workgroups in flight, and only the part of the tail
        // that is needed, by the split that needs it.  us in a graph, caches cold, 8 waves / 4: 16 rows x 24 heads of 64, 750 tokens
        // 16.1 / 16.0 (bf16 15.1 / 13.9), 64 rows 45 / 38, 8 rows x 16 heads x 200 tokens 7.9 / 9.2, 16 x 16 x 700 11.2 / 12.5; tail early /
        // late: 64 rows x 200 tokens f32 28.0 / 22.8, 2 rows x 16 heads x 700 tokens 8.4 / 9.1
        const long long wgs = (long long)grid.x * grid.y * grid.z;
        const bool early = a.splits == 1 && wgs <= 256, wide = cache->hd <= 64 && wgs <= 256;
        const unsigned g1 = (unsigned)qtiles | (unsigned)a.q_bf16 << 16 | (unsigned)(cache->tail_dtype == ACMI_BF16) << 17 | (unsigned)d.len_stride << 18 |
                            (unsigned)early << 19;
#define KV8_SPLIT_NW(HDv, Q, P, NWv)                                                                                                              \
    hipLaunchKernelGGL((kv8_attn_split_kernel<HDv, Q, P, NWv>), grid, dim3(NWv * 64), 0, st, a.q, a.len, cache->k_tail, cache->v_tail, g0, g1,        \
                       (int)d.q_row, d.S > 1 ? (int)d.q_tok : 0, (int)d.q_head, d.S, a)
#define KV8_SPLIT(HDv, Q, P)                                               \
    if (wide) KV8_SPLIT_NW(HDv, Q, P, (HDv <= 64 ? 8 : 4));               \
    else KV8_SPLIT_NW(HDv, Q, P, 4)
#define KV8_CASE(HDv)                                            \
    case HDv:                                                    \
        if (out_f32) { KV8_SPLIT(HDv, true, true); }             \
        else if (qhl) { KV8_SPLIT(HDv, true, false); }           \
        else { KV8_SPLIT(HDv, false, false); }                   \
        break;
        KV8_HD_SWITCH(cache->hd, KV8_CASE)
#undef KV8_CASE
#undef KV8_SPLIT
#undef KV8_SPLIT_NW
        if (int rc = acmi_check_launch("kv8_attn_split_kernel")) return rc;
        if (a.splits == 1) return ACMI_OK;
        const dim3 jgrid(min(d.S * a.G, 16), cache->H * qtiles, cache->rows);
#define KV8_CASE(HDv) case HDv: hipLaunchKernelGGL((kv8_attn_join_kernel<HDv>), jgrid, dim3(256), 0, st, a); break;
        KV8_HD_SWITCH(cache->hd, KV8_CASE)
#undef KV8_CASE
        return acmi_check_launch("kv8_attn_join_kernel");
    }
    const long long pairs = ((long long)cache->rows * cache->H + 7) / 8 * 8;
    // two column tiles per wave where bf16 results at 64 features leave the registers for it and the workgroups still fill the chip,
    // three per CU.  Measured, us one / two: 4 x 16 heads x 4096 tokens (2048 workgroups of two) 246 / 228, 16 x 24 x 600 (1920)
    // 52.3 / 53.0, 8 x 8 x 4 x 512 of 2048 (1024) 110 / 105; 16 x 16 x 100 of 1500 (256) 32.6 / 40.8; f32 results and 32 features, where
    // tried, gained nothing (4 x 16 x 4096 341 / 344, 8 x 16 x 2048 101 / 100)
    const int QB = cache->hd == 64 && !out_f32 && !qhl && pairs * ((qtiles + 7) / 8) >= 768 ? 2 : 1;
    a.tiles = (qtiles + 4 * QB - 1) / (4 * QB);
    a.splits = a.chunk = 1;   // (kv8_span divides by them)
    ACMI_REQUIRE(pairs * a.tiles * 256 <= 0xffffffffLL, "acmi_kv8_attn: %lld workgroups (a launch counts its work items in 32 bits)", pairs * a.tiles);
    const dim3 mgrid((unsigned)(pairs * a.tiles));
#define KV8_MANY(HDv, Q, P, QBv) hipLaunchKernelGGL((kv8_attn_many_kernel<HDv, Q, P, QBv>), mgrid, dim3(256), 0, st, a)
#define KV8_CASE(HDv)                                            \
    case HDv:                                                    \
        if (out_f32) KV8_MANY(HDv, true, true, 1);               \
        else if (qhl) KV8_MANY(HDv, true, false, 1);             \
        else if (QB == 1) KV8_MANY(HDv, false, false, 1);        \
        else KV8_MANY(64, false, false, 2);                      \
        break;
    KV8_HD_SWITCH(cache->hd, KV8_CASE)
#undef KV8_CASE
#undef KV8_MANY
    return acmi_check_launch("kv8_attn_many_kernel");
}
