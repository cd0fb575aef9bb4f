// Key / value cache in 8 bits and the attention over it, gfx950 (CDNA4, wave64).  Format: include/acmi.h (acmi_kv8_cache).
// Reference semantics: audiocraft/modules/transformer.py:266-298 (_complete_kv), :412-414 (scaled_dot_product_attention).
#include "acmi_lm_internal.h"

#include <math.h>

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
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
// place of token t inside a block's 64 bytes of one value feature (include/acmi.h)
__device__ __forceinline__ int kv8_vplace(int t) { return ((t >> 2) & 3) * 16 + (t >> 4) * 4 + (t & 3); }

// =====================================================================================================
// quantising a block
// =====================================================================================================
// 256 threads, hd / 16 rounds: thread chunk e = 16 consecutive features of a token (keys), resp. the 16 tokens of one lane group of
// a feature (values), so that every code store is 16 bytes.  get(which, token, feature) returns the value as the tail holds it.
__device__ __forceinline__ uint32_t kv8_code(float x, float inv) { return (uint32_t)(uint8_t)(int8_t)(int)rintf(x * inv); }

struct Kv8Scale { float scale, inv; };
__device__ __forceinline__ Kv8Scale kv8_scale(float amax, bool bad) {   // bad: a NaN or an infinity among the values
    Kv8Scale s;
    if (bad) { s.scale = __uint_as_float(0x7fc00000u); s.inv = 0.f; }
    else if (amax < 7.52316384526264e-37f) { s.scale = 0.f; s.inv = 0.f; }   // 2^-120: 127 / amax stays finite above
    else { s.scale = __fdiv_rn(amax, 127.f); s.inv = __fdiv_rn(127.f, amax); }
    return s;
}
// (amax, bad) over the workgroup of 256 threads: +infinity marks bad
__device__ __forceinline__ float kv8_block_max(float v, float* red) {
    v = wave_max(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    __syncthreads();
    return v;
}

template <int HD, typename G>
__device__ __forceinline__ void kv8_quantise_block(const acmi_kv8_cache& c, int row, int h, int blk, float* red, const G& get) {
    constexpr int RND = HD >= 64 ? HD / 64 : 1;            // rounds of 256 chunks of 16 elements
    constexpr int NCH = HD * BLK / 16;                     // chunks
    const size_t hb = ((size_t)row * c.H + h) * c.nblk + blk;
    float x[RND][16];
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        float amax = 0.f;
#pragma unroll
        for (int q = 0; q < RND; ++q) {
            const int ch = q * 256 + threadIdx.x;
            if (ch < NCH) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    if (part == 0) x[q][j] = get(0, ch / (HD / 16), ch % (HD / 16) * 16 + j);
                    else x[q][j] = get(1, (j >> 2) * 16 + (ch / HD) * 4 + (j & 3), ch % HD);
                    // NaN: fmaxf would drop it
                    amax = fmaxf(amax, isfinite(x[q][j]) ? fabsf(x[q][j]) : INFINITY);
                }
            }
        }
        amax = kv8_block_max(amax, red);
        const Kv8Scale s = kv8_scale(amax, amax == INFINITY);
        if (threadIdx.x == 0) (part == 0 ? c.k_scale : c.v_scale)[hb] = s.scale;
        uint8_t* dst = reinterpret_cast<uint8_t*>(part == 0 ? c.k_codes : c.v_codes) + hb * (size_t)(BLK * HD);
#pragma unroll
        for (int q = 0; q < RND; ++q) {
            const int ch = q * 256 + threadIdx.x;
            if (ch < NCH) {
                u32x4 w;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    w[k] = kv8_code(x[q][4 * k], s.inv) | kv8_code(x[q][4 * k + 1], s.inv) << 8 |
                           kv8_code(x[q][4 * k + 2], s.inv) << 16 | kv8_code(x[q][4 * k + 3], s.inv) << 24;
                const size_t at = part == 0 ? (size_t)ch * 16 : (size_t)(ch % HD) * BLK + (ch / HD) * 16;
                *reinterpret_cast<u32x4*>(dst + at) = w;
            }
        }
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
    __shared__ float red[4];
    const int j = blockIdx.x, h = blockIdx.y, row = blockIdx.z;
    const int cap = p.c.nblk * BLK, tb = p.c.tail_dtype == ACMI_BF16;
    const int start = p.start[row];
    const int n = min(p.n != nullptr ? p.n[row] : p.L, p.L);
    if (start < 0 || start >= cap || n <= 0) return;
    const int end = (int)min((long long)start + n, (long long)cap);
    const int b0 = start / BLK, b1 = end / BLK, blk = b0 + j, last = (end - 1) / BLK;
    const size_t tbase = ((size_t)row * p.c.H + h) * (BLK * HD);
    const size_t kb = (size_t)(row * p.k_row + h * p.k_head), vb = (size_t)(row * p.v_row + h * p.v_head);
    if (blk < b1) {
        kv8_quantise_block<HD>(p.c, row, h, blk, red, [&](int part, int t, int d) {
            const int pos = blk * BLK + t;
            if (pos < start) return kv8_ld(part == 0 ? p.c.k_tail : p.c.v_tail, tbase + t * HD + d, tb);
            const size_t i = (part == 0 ? kb : vb) + (size_t)(pos - start) * (part == 0 ? p.k_tok : p.v_tok) + d;
            return kv8_round(kv8_ld(part == 0 ? p.k : p.v, i, p.bf16), tb);
        });
    }
    if (j == 0) {
        __syncthreads();   // the old tail has been read
        const int first = max(start, last * BLK);
        for (int e = threadIdx.x; e < (end - first) * HD; e += 256) {
            const int pos = first + e / HD, d = e % HD;
            const size_t at = tbase + (size_t)(pos % BLK) * HD + d;
            kv8_st(p.c.k_tail, at, tb, kv8_ld(p.k, kb + (size_t)(pos - start) * p.k_tok + d, p.bf16));
            kv8_st(p.c.v_tail, at, tb, kv8_ld(p.v, vb + (size_t)(pos - start) * p.v_tok + d, p.bf16));
        }
    }
}

// =====================================================================================================
// load
// =====================================================================================================
struct Kv8LoadArgs { acmi_kv8_cache c; const int* len; int T; void* k; void* v; int bf16; };

template <int HD>
__global__ __launch_bounds__(256) void kv8_load_kernel(const Kv8LoadArgs p) {
    const int blk = blockIdx.x, h = blockIdx.y, row = blockIdx.z;
    const int tb = p.c.tail_dtype == ACMI_BF16;
    const int len = min(p.len[row], p.c.nblk * BLK), last = max(len - 1, 0) / BLK;
    const size_t rh = (size_t)row * p.c.H + h, hb = rh * p.c.nblk + blk;
    const bool coded = blk < last;
    const float ks = coded ? p.c.k_scale[hb] : 0.f, vs = coded ? p.c.v_scale[hb] : 0.f;
    const int8_t* kc = reinterpret_cast<const int8_t*>(p.c.k_codes) + hb * (size_t)(BLK * HD);
    const int8_t* vc = reinterpret_cast<const int8_t*>(p.c.v_codes) + hb * (size_t)(BLK * HD);
    for (int e = threadIdx.x; e < BLK * HD; e += 256) {
        const int t = e / HD, d = e % HD, pos = blk * BLK + t;
        if (pos >= p.T) break;
        float k = 0.f, v = 0.f;
        if (pos < len) {
            if (coded) {
                k = (float)kc[t * HD + d] * ks;
                v = (float)vc[d * BLK + kv8_vplace(t)] * vs;
            } else {
                k = kv8_ld(p.c.k_tail, rh * (BLK * HD) + t * HD + d, tb);
                v = kv8_ld(p.c.v_tail, rh * (BLK * HD) + t * HD + d, tb);
            }
        }
        const size_t at = (rh * p.T + pos) * HD + d;
        kv8_st(p.k, at, p.bf16, k);
        kv8_st(p.v, at, p.bf16, v);
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
// The block's scales multiply the scores and the block's part of O.  Probabilities are carried as 2^14 p (f16 then resolves
// p down to 2^-38).  The newest block comes from the tail in f32 through the f32 matrix instruction, 16 tokens per wave.
struct Kv8AttnArgs {
    acmi_kv8_cache c;
    const void* q; int q_bf16; long long q_row, q_tok, q_head;
    int S, Hq, G;
    const int* len; int len_stride, len_bias; const int* q_len; const int* start_rows;
    int causal, past;
    const void* kn; const void* vn; int n_bf16; long long kn_row, kn_head, vn_row, vn_head;
    int complete;
    void* out; int out_mode, out_bf16, out_rbs, out_col0;
    float* work; int splits;
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

template <int HD> struct Kv8Geo {
    static constexpr int KW = HD >= 64 ? HD / 16 : 2;     // 32-bit words of K codes per lane and 16 tokens
    static constexpr int NK = KW / 2;                     // products of 32 features
    static constexpr int ND = HD / 16;                    // 16-feature tiles of O^T
};
// the feature that element j of a lane's B operand of product c stands for (hd 16: lanes kg >= 2 hold nothing)
template <int HD> __device__ __forceinline__ int kv8_qdim(int kg, int c, int j) {
    if (HD >= 64) return (c >> 1) * 64 + kg * 16 + (c & 1) * 8 + j;
    return kg * 8 + j;
}

template <int HD> struct Kv8Raw { uint32_t k[4][Kv8Geo<HD>::KW]; u32x4 v[Kv8Geo<HD>::ND]; float ks, vs; };

template <int HD, bool NT>
__device__ __forceinline__ void kv8_fetch(const uint8_t* kc, const uint8_t* vc, const float* ks, const float* vs, int blk, Kv8Raw<HD>& r) {
    const int lane = threadIdx.x & 63, nl = lane & 15, kg = lane >> 4;
    const uint8_t* kb = kc + (size_t)blk * (BLK * HD);
    const uint8_t* vb = vc + (size_t)blk * (BLK * HD);
    auto ld16 = [](const uint8_t* p) { return NT ? __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p)) : *reinterpret_cast<const u32x4*>(p); };
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    auto ld8 = [](const uint8_t* p) { return NT ? __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p)) : *reinterpret_cast<const u32x2*>(p); };
    r.ks = ks[blk]; r.vs = vs[blk];
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
        const uint8_t* row = kb + (tt * 16 + nl) * HD;
        if constexpr (HD >= 64) {
#pragma unroll
            for (int l = 0; l < HD / 64; ++l) {
                const u32x4 w = ld16(row + l * 64 + kg * 16);
#pragma unroll
                for (int e = 0; e < 4; ++e) r.k[tt][l * 4 + e] = w[e];
            }
        } else {
            const u32x2 w = ld8(row + (HD == 32 ? kg : (kg & 1)) * 8);
            // hd 16: lanes kg >= 2 have no feature; their queries are 0, any code will do
            r.k[tt][0] = w[0]; r.k[tt][1] = w[1];
        }
    }
#pragma unroll
    for (int i = 0; i < Kv8Geo<HD>::ND; ++i) r.v[i] = ld16(vb + (i * 16 + nl) * BLK + kg * 16);
}

// one column tile's state: lane (kg, n) belongs to column n
template <int HD, bool QHL> struct Kv8Col {
    f16x8 qh[Kv8Geo<HD>::NK], ql[QHL ? Kv8Geo<HD>::NK : 1];
    float sfac;          // score factor: softmax scale * log2(e) * the query's power of two
    int lo, lim;         // positions [lo, lim) are seen
    float m, l;
    f32x4 o[Kv8Geo<HD>::ND];
};

constexpr float KV8_PSHIFT = 14.f;

// scores s (log2 units, masked) of 16 * NT tokens -> probabilities * 2^14; returns the factor of the old sums
template <int NTT>
__device__ __forceinline__ float kv8_softmax(f32x4 (&s)[NTT], float& m, float& l, bool& none) {
    float cmax = -INFINITY;
#pragma unroll
    for (int tt = 0; tt < NTT; ++tt)
#pragma unroll
        for (int r = 0; r < 4; ++r) cmax = fmaxf(cmax, s[tt][r]);
    cmax = fmaxf(cmax, __shfl_xor(cmax, 16, 64));
    cmax = fmaxf(cmax, __shfl_xor(cmax, 32, 64));
    none = cmax == -INFINITY;
    const float m_new = fmaxf(m, cmax);
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m - m_use);
    const float base = m_use - KV8_PSHIFT;
    float sum = 0.f;
#pragma unroll
    for (int tt = 0; tt < NTT; ++tt)
#pragma unroll
        for (int r = 0; r < 4; ++r) { s[tt][r] = __builtin_amdgcn_exp2f(s[tt][r] - base); sum += s[tt][r]; }
    l = fmaf(l, alpha, sum);
    m = m_new;
    return alpha;
}

// a block of codes into one column tile
template <int HD, bool QHL, bool PHL>
__device__ __forceinline__ void kv8_block(Kv8Col<HD, QHL>& c, const f16x8 (&kf)[4][Kv8Geo<HD>::NK], const f16x8 (&vf)[Kv8Geo<HD>::ND][2],
                                          float ks, float vs, int t0) {
    constexpr int NK = Kv8Geo<HD>::NK, ND = Kv8Geo<HD>::ND;
    const int kg = (threadIdx.x & 63) >> 4;
    f32x4 s[4];
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
        s[tt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            s[tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[tt][k], c.qh[k], s[tt], 0, 0, 0);
            if constexpr (QHL) s[tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[tt][k], c.ql[k], s[tt], 0, 0, 0);
        }
    }
    const float f = ks * c.sfac;
    const bool all = c.lo <= t0 && c.lim >= t0 + BLK;
    if (__all(all)) {
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[tt][r] *= f;
    } else {
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = t0 + tt * 16 + kg * 4 + r;
                s[tt][r] = (t >= c.lo && t < c.lim) ? s[tt][r] * f : -INFINITY;
            }
    }
    bool none;
    const float alpha = kv8_softmax<4>(s, c.m, c.l, none);
    const float vse = none ? 0.f : vs;   // (a block poisoned by a NaN leaves columns that do not see it alone)
    f16x8 ph[2], pl[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float a = s[2 * u + (e >> 1)][(e & 1) * 2], b = s[2 * u + (e >> 1)][(e & 1) * 2 + 1];
            const f16x2 h = kv8_pk(a, b);
            ph[u][2 * e] = h[0]; ph[u][2 * e + 1] = h[1];
            if constexpr (PHL) {
                const f16x2 w = kv8_pk(a - (float)h[0], b - (float)h[1]);
                pl[u][2 * e] = w[0]; pl[u][2 * e + 1] = w[1];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < ND; ++i) {
        f32x4 t = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            t = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[i][u], ph[u], t, 0, 0, 0);
            if constexpr (PHL) t = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[i][u], pl[u], t, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) c.o[i][r] = fmaf(t[r], vse, c.o[i][r] * alpha);
    }
}

template <int HD>
__device__ __forceinline__ void kv8_convert(const Kv8Raw<HD>& r, f16x8 (&kf)[4][Kv8Geo<HD>::NK], f16x8 (&vf)[Kv8Geo<HD>::ND][2]) {
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int k = 0; k < Kv8Geo<HD>::NK; ++k) kf[tt][k] = kv8_cvt(r.k[tt][2 * k], r.k[tt][2 * k + 1]);
#pragma unroll
    for (int i = 0; i < Kv8Geo<HD>::ND; ++i) {
        vf[i][0] = kv8_cvt(r.v[i][0], r.v[i][1]);
        vf[i][1] = kv8_cvt(r.v[i][2], r.v[i][3]);
    }
}

// what a column is: row geometry shared by both kernels
struct Kv8RowInfo { int len, qlen, start; bool fresh; };   // fresh: the call brings the row's newest token (and it fits)
__device__ __forceinline__ Kv8RowInfo kv8_row(const Kv8AttnArgs& p, int row) {
    Kv8RowInfo r;
    const long long len = (long long)p.len[(size_t)row * p.len_stride] + p.len_bias;
    r.len = (int)max(0LL, min(len, (long long)p.c.nblk * BLK));
    r.fresh = p.kn != nullptr && r.len == len && len > 0;
    r.qlen = p.q_len != nullptr ? max(0, min(p.q_len[row], p.S)) : p.S;
    r.start = p.start_rows != nullptr ? max(0, p.start_rows[row]) : 0;
    return r;
}

// column c of (row, cache head): visible range and query; cidx may lie past the last column
template <int HD, bool QHL>
__device__ __forceinline__ void kv8_column(const Kv8AttnArgs& p, const Kv8RowInfo& ri, int row, int kvh, int cidx, Kv8Col<HD, QHL>& c) {
    const int kg = (threadIdx.x & 63) >> 4;
    const int s = cidx / p.G, g = cidx - s * p.G;
    const bool live = s < ri.qlen;
    const int pos = ri.len - ri.qlen + s;
    // (columns without a query are never stored: they see everything, so that they do not keep a block on the masked path)
    c.lim = !live ? 0x7fffffff : p.causal ? max(0, min(pos + 1, ri.len)) : ri.len;
    c.lo = live ? ri.start : 0;
    if (live && p.causal && p.past > 0) c.lo = max(c.lo, pos - p.past);
    if (c.lo >= c.lim) { c.lo = 0; c.lim = 0; }
    c.m = -INFINITY; c.l = 0.f;
#pragma unroll
    for (int i = 0; i < Kv8Geo<HD>::ND; ++i) c.o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float x[Kv8Geo<HD>::NK][8], amax = 0.f;
    const long long qb = row * p.q_row + (long long)s * p.q_tok + (long long)(kvh * p.G + g) * p.q_head;
#pragma unroll
    for (int k = 0; k < Kv8Geo<HD>::NK; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int d = kv8_qdim<HD>(kg, k, j);
            x[k][j] = (live && d < HD) ? kv8_ld(p.q, (size_t)(qb + d), p.q_bf16) : 0.f;
            amax = fmaxf(amax, isfinite(x[k][j]) ? fabsf(x[k][j]) : INFINITY);
        }
    amax = fmaxf(amax, __shfl_xor(amax, 16, 64));
    amax = fmaxf(amax, __shfl_xor(amax, 32, 64));
    // x = xn * 2^(e - 14) with the largest |xn| in [2^14, 2^15); a query with a NaN or an infinity gives NaN
    const int e = (amax > 0.f && amax < INFINITY) ? ilogbf(amax) : 0;
    const float down = ldexpf(1.f, 14 - e < 127 ? 14 - e : 127);   // (features below 2^-113 all over: the product below stays exact)
    c.sfac = amax == INFINITY ? __uint_as_float(0x7fc00000u) : p.scale * 1.4426950408889634f / down;
#pragma unroll
    for (int k = 0; k < Kv8Geo<HD>::NK; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float y = amax == INFINITY ? 0.f : x[k][j] * down;
            const _Float16 h = (_Float16)y;
            c.qh[k][j] = h;
            if constexpr (QHL) c.ql[k][j] = (_Float16)(y - (float)h);
        }
}

// 16 tokens (slot0 ..) of the tail into one column tile, in f32.  last: the tail's block
template <int HD, bool QHL>
__device__ __forceinline__ void kv8_tail(const Kv8AttnArgs& p, const Kv8RowInfo& ri, int row, int kvh, int cidx, int slot0, Kv8Col<HD, QHL>& c) {
    constexpr int ND = Kv8Geo<HD>::ND;
    const int lane = threadIdx.x & 63, nl = lane & 15, kg = lane >> 4;
    const int last = (ri.len - 1) / BLK, t0 = last * BLK + slot0, tb = p.c.tail_dtype == ACMI_BF16;
    if (t0 >= ri.len) return;   // (wave uniform)
    const size_t base = ((size_t)row * p.c.H + kvh) * (BLK * HD);
    const int s_ = cidx / p.G, g = cidx - s_ * p.G;
    const bool live = s_ < ri.qlen;
    const long long qb = row * p.q_row + (long long)s_ * p.q_tok + (long long)(kvh * p.G + g) * p.q_head;
    auto val = [&](int part, int t, int d) {   // t: position; past the row's length: 0
        if (t >= ri.len) return 0.f;
        if (ri.fresh && t == ri.len - 1) {
            const long long i = (part == 0 ? row * p.kn_row + kvh * p.kn_head : row * p.vn_row + kvh * p.vn_head) + d;
            return kv8_round(kv8_ld(part == 0 ? p.kn : p.vn, (size_t)i, p.n_bf16), tb);
        }
        return kv8_ld(part == 0 ? p.c.k_tail : p.c.v_tail, base + (size_t)(t - last * BLK) * HD + d, tb);
    };
    f32x4 s[1] = {f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int d = i * 16 + kg * 4 + j;
            const float a = val(0, t0 + nl, d);
            const float b = live ? kv8_ld(p.q, (size_t)(qb + d), p.q_bf16) : 0.f;
            s[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, s[0], 0, 0, 0);
        }
    const float f = p.scale * 1.4426950408889634f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int t = t0 + kg * 4 + r;
        s[0][r] = (t >= c.lo && t < c.lim) ? s[0][r] * f : -INFINITY;
    }
    bool none;
    const float alpha = kv8_softmax<1>(s, c.m, c.l, none);
    bool bad = false;   // a NaN or an infinity among the values: it must not meet the probability 0 of a column that does not see it
#pragma unroll
    for (int i = 0; i < ND; ++i) {
        f32x4 t = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float v = val(1, t0 + kg * 4 + r, i * 16 + nl);
            const bool fin = isfinite(v);
            bad |= !fin;
            t = __builtin_amdgcn_mfma_f32_16x16x4f32(fin ? v : 0.f, s[0][r], t, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) c.o[i][r] = fmaf(c.o[i][r], alpha, t[r]);
    }
    if (__any(bad)) {   // those values one by one, each column for itself
        for (int tok = 0; tok < 16; ++tok) {
            float pr = 0.f;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float x = __shfl(s[0][r], (tok >> 2) * 16 + nl, 64);
                if ((tok & 3) == r) pr = x;
            }
            const int t = t0 + tok;
            const bool seen = t >= c.lo && t < c.lim;
#pragma unroll
            for (int i = 0; i < ND; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float v = val(1, t, i * 16 + kg * 4 + r);
                    if (seen && !isfinite(v)) c.o[i][r] = fmaf(pr, v, c.o[i][r]);
                }
        }
    }
}

// the blocks of codes a column tile visits, and how many workgroups share them
struct Kv8Span { int bf, bt, eff; bool live, tail; };
constexpr int KV8_MIN_BLOCKS = 8;   // blocks per workgroup below which no further split is made
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
    s.eff = max(1, min(p.splits, (s.bt - s.bf) / KV8_MIN_BLOCKS));
    s.tail = lim > nf * BLK && lo < ri.len;
    return s;
}

// out of a finished column: 4 consecutive features
__device__ __forceinline__ void kv8_put4(const Kv8AttnArgs& p, int row, int s, int head, int HD, int d, const f32x4& v) {
    const size_t at = (((size_t)row * p.S + s) * p.Hq + head) * HD + d;
    if (p.out_mode == ACMI_OUT_F32) *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p.out) + at) = v;
    else if (p.out_mode == ACMI_OUT_BF16)
        *reinterpret_cast<uint2*>(reinterpret_cast<bf16_t*>(p.out) + at) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    else {
        const int col = p.out_col0 + head * HD + d;   // (a multiple of 4: the four features share a lane's 16 bytes)
        if (p.out_bf16)
            *reinterpret_cast<uint2*>(reinterpret_cast<bf16_t*>(p.out) + tiled_index<bf16_t>(row, col, p.out_rbs)) =
                make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
        else *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p.out) + tiled_index<float>(row, col, p.out_rbs)) = v;
    }
}

// ---- few queries: one workgroup per (column tile, cache head, row, split); its four waves take the blocks in turn and 16 tokens
// of the tail each, and are joined through LDS
template <int HD, bool QHL, bool PHL>
__global__ __launch_bounds__(256) void kv8_attn_split_kernel(const Kv8AttnArgs p) {
    constexpr int ND = Kv8Geo<HD>::ND, PITCH = HD + 4;
    __shared__ __attribute__((aligned(16))) float sm_o[4][16][PITCH];
    __shared__ float sm_m[4][16], sm_l[4][16], red[4];
    const int split = blockIdx.x, row = blockIdx.z;
    const int qtiles = (p.S * p.G + 15) / 16, kvh = blockIdx.y / qtiles, qt = blockIdx.y - kvh * qtiles;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nl = lane & 15, kg = lane >> 4;
    const Kv8RowInfo ri = kv8_row(p, row);
    const Kv8Span sp = kv8_span(p, ri, qt * 16, min(qt * 16 + 16, p.S * p.G));
    if (split >= sp.eff) return;
    const int per = (sp.bt - sp.bf + sp.eff - 1) / sp.eff;
    const int s0 = sp.bf + split * per, s1 = min(sp.bt, s0 + per);
    const size_t rh = (size_t)row * p.c.H + kvh, hb = rh * p.c.nblk;
    const uint8_t* kc = reinterpret_cast<const uint8_t*>(p.c.k_codes) + hb * (BLK * HD);
    const uint8_t* vc = reinterpret_cast<const uint8_t*>(p.c.v_codes) + hb * (BLK * HD);
    const float* ks = p.c.k_scale + hb; const float* vs = p.c.v_scale + hb;

    Kv8Col<HD, QHL> c;
    Kv8Raw<HD> ra, rb;
    int b = s0 + wave;
    if (b < s1) kv8_fetch<HD, true>(kc, vc, ks, vs, b, ra);
    kv8_column<HD, QHL>(p, ri, row, kvh, qt * 16 + nl, c);
    const bool mine = split == sp.eff - 1;   // the split that owns the tail
    if (mine && sp.tail) kv8_tail<HD, QHL>(p, ri, row, kvh, qt * 16 + nl, wave * 16, c);
    f16x8 kf[4][Kv8Geo<HD>::NK], vf[ND][2];
    while (b < s1) {   // two raw blocks in flight
        if (b + 4 < s1) kv8_fetch<HD, true>(kc, vc, ks, vs, b + 4, rb);
        kv8_convert<HD>(ra, kf, vf);
        kv8_block<HD, QHL, PHL>(c, kf, vf, ra.ks, ra.vs, b * BLK);
        b += 4;
        if (b >= s1) break;
        if (b + 4 < s1) kv8_fetch<HD, true>(kc, vc, ks, vs, b + 4, ra);
        kv8_convert<HD>(rb, kf, vf);
        kv8_block<HD, QHL, PHL>(c, kf, vf, rb.ks, rb.vs, b * BLK);
        b += 4;
    }
    float l = c.l;
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
#pragma unroll
    for (int i = 0; i < ND; ++i) *reinterpret_cast<f32x4*>(&sm_o[wave][nl][i * 16 + kg * 4]) = c.o[i];
    if (kg == 0) { sm_m[wave][nl] = c.m; sm_l[wave][nl] = l; }
    // the row's newest token and a block it completes (column tile 0 alone)
    if (mine && qt == 0 && ri.len > 0 && (ri.fresh || p.complete)) {
        const int last = (ri.len - 1) / BLK, tb = p.c.tail_dtype == ACMI_BF16;
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
        if (ri.len % BLK == 0)
            kv8_quantise_block<HD>(p.c, row, kvh, last, red, [&](int part, int t, int d) {
                if (t == BLK - 1 && ri.fresh) return kv8_round(newest(part, d), tb);
                return kv8_ld(part == 0 ? p.c.k_tail : p.c.v_tail, tbase + t * HD + d, tb);
            });
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 16 * HD / 4; e += 256) {
        const int n = e / (HD / 4), d = e % (HD / 4) * 4, cidx = qt * 16 + n;
        if (cidx >= p.S * p.G) continue;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) M = fmaxf(M, sm_m[w][n]);
        const float Mu = M == -INFINITY ? 0.f : M;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        float den = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = __builtin_amdgcn_exp2f(sm_m[w][n] - Mu);
            const f32x4 x = *reinterpret_cast<const f32x4*>(&sm_o[w][n][d]);
            den = fmaf(f, sm_l[w][n], den);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = fmaf(f, x[r], o[r]);
        }
        if (sp.eff == 1) {
            const int s = cidx / p.G, g = cidx - s * p.G;
            const bool none = s >= ri.qlen || den == 0.f;
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = none ? 0.f : o[r] / den;
            kv8_put4(p, row, s, kvh * p.G + g, HD, d, o);
        } else {   // partial: [row][cache head x tile][split][column][features | max | sum]
            float* w = p.work + ((((size_t)row * gridDim.y + blockIdx.y) * p.splits + split) * 16 + n) * (HD + 4);
            *reinterpret_cast<f32x4*>(w + d) = o;
            if (d == 0) { w[HD] = M; w[HD + 1] = den; }
        }
    }
}

// joins the splits, in their order
template <int HD>
__global__ __launch_bounds__(256) void kv8_attn_join_kernel(const Kv8AttnArgs p) {
    const int row = blockIdx.y, qtiles = (p.S * p.G + 15) / 16, kvh = blockIdx.x / qtiles, qt = blockIdx.x - kvh * qtiles;
    const Kv8RowInfo ri = kv8_row(p, row);
    const Kv8Span sp = kv8_span(p, ri, qt * 16, min(qt * 16 + 16, p.S * p.G));
    if (sp.eff == 1) return;   // the split kernel has written it
    const float* base = p.work + ((size_t)row * gridDim.x + blockIdx.x) * p.splits * 16 * (HD + 4);
    for (int e = threadIdx.x; e < 16 * HD / 4; e += 256) {
        const int n = e / (HD / 4), d = e % (HD / 4) * 4, cidx = qt * 16 + n;
        if (cidx >= p.S * p.G) continue;
        const float* w = base + n * (HD + 4);
        float M = -INFINITY;
        for (int k = 0; k < sp.eff; ++k) M = fmaxf(M, w[(size_t)k * 16 * (HD + 4) + HD]);
        const float Mu = M == -INFINITY ? 0.f : M;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        float den = 0.f;
        for (int k = 0; k < sp.eff; ++k) {
            const float* x = w + (size_t)k * 16 * (HD + 4);
            const float f = __builtin_amdgcn_exp2f(x[HD] - Mu);
            const f32x4 v = *reinterpret_cast<const f32x4*>(x + d);
            den = fmaf(f, x[HD + 1], den);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = fmaf(f, v[r], o[r]);
        }
        const int s = cidx / p.G, g = cidx - s * p.G;
        const bool none = s >= ri.qlen || den == 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = none ? 0.f : o[r] / den;
        kv8_put4(p, row, s, kvh * p.G + g, HD, d, o);
    }
}

// ---- many queries: a wave owns QB column tiles and walks every block they see
template <int HD, bool QHL, bool PHL, int QB>
__global__ __launch_bounds__(256) void kv8_attn_many_kernel(const Kv8AttnArgs p) {
    constexpr int ND = Kv8Geo<HD>::ND;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nl = lane & 15, kg = lane >> 4;
    const int kvh = blockIdx.y, row = blockIdx.z, cols = p.S * p.G;
    const int c0 = (blockIdx.x * 4 + wave) * 16 * QB;
    if (c0 >= cols) return;
    const Kv8RowInfo ri = kv8_row(p, row);
    const Kv8Span sp = kv8_span(p, ri, c0, min(c0 + 16 * QB, cols));
    Kv8Col<HD, QHL> c[QB];
#pragma unroll
    for (int g = 0; g < QB; ++g) kv8_column<HD, QHL>(p, ri, row, kvh, c0 + g * 16 + nl, c[g]);
    if (sp.live) {
        const size_t rh = (size_t)row * p.c.H + kvh, hb = rh * p.c.nblk;
        const uint8_t* kc = reinterpret_cast<const uint8_t*>(p.c.k_codes) + hb * (BLK * HD);
        const uint8_t* vc = reinterpret_cast<const uint8_t*>(p.c.v_codes) + hb * (BLK * HD);
        for (int b = sp.bf; b < sp.bt; ++b) {
            Kv8Raw<HD> r;
            kv8_fetch<HD, false>(kc, vc, p.c.k_scale + hb, p.c.v_scale + hb, b, r);
            f16x8 kf[4][Kv8Geo<HD>::NK], vf[ND][2];
            kv8_convert<HD>(r, kf, vf);
#pragma unroll
            for (int g = 0; g < QB; ++g) kv8_block<HD, QHL, PHL>(c[g], kf, vf, r.ks, r.vs, b * BLK);
        }
        if (sp.tail)
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int g = 0; g < QB; ++g) kv8_tail<HD, QHL>(p, ri, row, kvh, c0 + g * 16 + nl, t * 16, c[g]);
    }
#pragma unroll
    for (int g = 0; g < QB; ++g) {
        float l = c[g].l;
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        const int cidx = c0 + g * 16 + nl, s = cidx / p.G, h = cidx - s * p.G;
        if (cidx >= cols) continue;
        const bool none = s >= ri.qlen || l == 0.f;
#pragma unroll
        for (int i = 0; i < ND; ++i) {
            f32x4 o;
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = none ? 0.f : c[g].o[i][r] / l;
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
    ACMI_REQUIRE(c->rows > 0 && c->rows <= 65535 && c->H > 0 && c->H <= 65535 && c->nblk > 0 && c->nblk <= (1 << 24),
                 "%s: bad cache shape rows=%d H=%d nblk=%d", who, c->rows, c->H, c->nblk);
    ACMI_REQUIRE(c->tail_dtype == ACMI_F32 || c->tail_dtype == ACMI_BF16, "%s: tail_dtype %d", who, c->tail_dtype);
    ACMI_REQUIRE(c->k_codes && c->v_codes && c->k_scale && c->v_scale && c->k_tail && c->v_tail, "%s: null cache buffer", who);
    return ACMI_OK;
}
static bool kv8_dtype_ok(int d) { return d == ACMI_F32 || d == ACMI_BF16; }

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
    ACMI_REQUIRE(desc != nullptr && desc->start != nullptr, "acmi_kv8_store: null descriptor or start");
    ACMI_REQUIRE(desc->L >= 0 && desc->L <= (1 << 30) && kv8_dtype_ok(desc->dtype), "acmi_kv8_store: L=%d dtype=%d", desc->L, desc->dtype);
    if (desc->L == 0) return ACMI_OK;
    ACMI_REQUIRE(desc->k && desc->v, "acmi_kv8_store: null k or v");
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
    ACMI_REQUIRE(k_out && v_out, "acmi_kv8_load: null output");
    Kv8LoadArgs a = {};
    a.c = *cache; a.len = len; a.T = T; a.k = k_out; a.v = v_out; a.bf16 = out_dtype == ACMI_BF16;
    const dim3 grid((T + BLK - 1) / BLK, cache->H, cache->rows);
#define KV8_CASE(HDv) case HDv: hipLaunchKernelGGL((kv8_load_kernel<HDv>), grid, dim3(256), 0, (hipStream_t)stream, a); break;
    KV8_HD_SWITCH(cache->hd, KV8_CASE)
#undef KV8_CASE
    return acmi_check_launch("kv8_load_kernel");
}

// column tiles up to which the split form runs
constexpr int KV8_SPLIT_TILES = 4;
static bool kv8_few(int S, int G) { return (S * G + 15) / 16 <= KV8_SPLIT_TILES; }
static int kv8_splits(const acmi_kv8_cache* c, int S, int G) {
    const long long wgs = (long long)c->rows * c->H * ((S * G + 15) / 16);
    const long long want = (1024 + wgs - 1) / wgs, most = c->nblk / KV8_MIN_BLOCKS;
    return (int)max(1LL, min(min(want, most), 64LL));
}

extern "C" size_t acmi_kv8_attn_work_floats(const acmi_kv8_cache* cache, int S, int Hq) {
    if (kv8_check(cache, "acmi_kv8_attn_work_floats") || S <= 0 || Hq <= 0 || Hq % cache->H) return 0;
    const int G = Hq / cache->H;
    if (!kv8_few(S, G)) return 0;
    const int sp = kv8_splits(cache, S, G);
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
    ACMI_REQUIRE(d.past_context >= 0 && (d.past_context == 0 || d.causal), "acmi_kv8_attn: past_context=%d needs causal", d.past_context);
    Kv8AttnArgs a = {};
    a.c = *cache; a.q = d.q; a.q_bf16 = d.q_dtype == ACMI_BF16; a.q_row = d.q_row; a.q_tok = d.q_tok; a.q_head = d.q_head;
    a.S = d.S; a.Hq = d.Hq; a.G = d.Hq / cache->H;
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
    const bool qhl = d.q_dtype == ACMI_F32;   // (a bf16 query is one f16 exactly)
    hipStream_t st = (hipStream_t)stream;
    const int qtiles = (d.S * a.G + 15) / 16;
    if (kv8_few(d.S, a.G)) {
        a.splits = kv8_splits(cache, d.S, a.G);
        a.work = d.work;
        ACMI_REQUIRE(a.splits == 1 || (d.work != nullptr && (reinterpret_cast<size_t>(d.work) & 15) == 0),
                     "acmi_kv8_attn: needs acmi_kv8_attn_work_floats floats of 16-byte aligned work");
        ACMI_REQUIRE((long long)cache->H * qtiles <= 65535, "acmi_kv8_attn: %d heads x %d column tiles", cache->H, qtiles);
        const dim3 grid(a.splits, cache->H * qtiles, cache->rows);
#define KV8_SPLIT(HDv, Q, P) hipLaunchKernelGGL((kv8_attn_split_kernel<HDv, Q, P>), grid, dim3(256), 0, st, a)
#define KV8_CASE(HDv)                                                       \
    case HDv:                                                               \
        if (qhl) { if (out_f32) KV8_SPLIT(HDv, true, true); else KV8_SPLIT(HDv, true, false); }   \
        else { if (out_f32) KV8_SPLIT(HDv, false, true); else KV8_SPLIT(HDv, false, false); }     \
        break;
        KV8_HD_SWITCH(cache->hd, KV8_CASE)
#undef KV8_CASE
#undef KV8_SPLIT
        if (int rc = acmi_check_launch("kv8_attn_split_kernel")) return rc;
        if (a.splits == 1) return ACMI_OK;
        const dim3 jgrid(cache->H * qtiles, cache->rows);
#define KV8_CASE(HDv) case HDv: hipLaunchKernelGGL((kv8_attn_join_kernel<HDv>), jgrid, dim3(256), 0, st, a); break;
        KV8_HD_SWITCH(cache->hd, KV8_CASE)
#undef KV8_CASE
        return acmi_check_launch("kv8_attn_join_kernel");
    }
#define KV8_MANY(HDv, Q, P, QBv)                                                                                             \
    hipLaunchKernelGGL((kv8_attn_many_kernel<HDv, Q, P, QBv>), dim3((qtiles + 4 * QBv - 1) / (4 * QBv), cache->H, cache->rows), dim3(256), 0, st, a)
#define KV8_CASE(HDv)                                                       \
    case HDv: {                                                             \
        constexpr int QBv = HDv <= 64 ? 2 : 1;                              \
        if (qhl) { if (out_f32) KV8_MANY(HDv, true, true, QBv); else KV8_MANY(HDv, true, false, QBv); }   \
        else { if (out_f32) KV8_MANY(HDv, false, true, QBv); else KV8_MANY(HDv, false, false, QBv); }     \
        break;                                                              \
    }
    KV8_HD_SWITCH(cache->hd, KV8_CASE)
#undef KV8_CASE
#undef KV8_MANY
    return acmi_check_launch("kv8_attn_many_kernel");
}
