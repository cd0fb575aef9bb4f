// Projection in 8-bit integers, gfx950 (CDNA4, wave64): rows quantised with a scale each (tokens of an activation, output
// channels of a weight), int8 x int8 products summed exactly in 32-bit integers by the matrix cores, one f32 scaling at the end.
// Format: include/acmi.h.  Reference semantics: the nn.Linear projections of audiocraft/modules/transformer.py:362-399, 454-574.
#include "acmi_lm_internal.h"

#include <math.h>

typedef int i32x4 __attribute__((ext_vector_type(4)));

// =====================================================================================================
// rows -> int8 fragments + a scale each
// =====================================================================================================
struct QuantRowsArgs { const void* x; int bf16; long long ldx; int R, K, nkc; uint8_t* codes; float* scale; };

__device__ __forceinline__ float i8_ld(const void* p, size_t i, int bf16) {
    return bf16 ? bf16_to_f32(reinterpret_cast<const bf16_t*>(p)[i]) : reinterpret_cast<const float*>(p)[i];
}
__device__ __forceinline__ uint32_t i8_code(float x, float inv) { return (uint32_t)(uint8_t)(int8_t)(int)rintf(x * inv); }

// one workgroup per row; a thread owns chunks of 16 consecutive columns = the 16 bytes of one lane of a fragment
__global__ __launch_bounds__(256) void quant_rows_kernel(const QuantRowsArgs p) {
    __shared__ float red[4];
    const int row = blockIdx.x, nch = p.nkc * 4;
    const size_t xb = (size_t)(row * p.ldx);
    float amax = 0.f;
    for (int k = threadIdx.x; k < p.K; k += 256) {
        const float v = i8_ld(p.x, xb + k, p.bf16);
        amax = fmaxf(amax, isfinite(v) ? fabsf(v) : INFINITY);   // (fmaxf would drop a NaN)
    }
    amax = wave_max(amax);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = amax;
    __syncthreads();
    amax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    float scale, inv;
    if (amax == INFINITY) { scale = __uint_as_float(0x7fc00000u); inv = 0.f; }
    else if (amax < 7.52316384526264e-37f) { scale = 0.f; inv = 0.f; }   // 2^-120
    else { scale = __fdiv_rn(amax, 127.f); inv = __fdiv_rn(127.f, amax); }
    if (threadIdx.x == 0) p.scale[row] = scale;
    for (int ch = threadIdx.x; ch < nch; ch += 256) {
        u32x4 w;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint32_t b = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int col = ch * 16 + k * 4 + e;
                const float v = col < p.K ? i8_ld(p.x, xb + col, p.bf16) : 0.f;
                b |= i8_code(v, inv) << (8 * e);
            }
            w[k] = b;
        }
        const size_t frag = (size_t)(row >> 4) * p.nkc + (ch >> 2);
        *reinterpret_cast<u32x4*>(p.codes + frag * 1024 + ((ch & 3) * 16 + (row & 15)) * 16) = w;
    }
}

extern "C" int acmi_quantize_rows_i8(const void* x, int dtype, long long ldx, int R, int K, void* codes, float* scale, void* stream) {
    ACMI_REQUIRE(dtype == ACMI_F32 || dtype == ACMI_BF16, "acmi_quantize_rows_i8: dtype %d", dtype);
    ACMI_REQUIRE(R >= 0 && K > 0 && K <= 131072, "acmi_quantize_rows_i8: R=%d K=%d (K in [1, 131072])", R, K);
    if (R == 0) return ACMI_OK;
    ACMI_REQUIRE(x && codes && scale && ldx >= K, "acmi_quantize_rows_i8: null buffer or ldx=%lld < K=%d", ldx, K);
    ACMI_REQUIRE((reinterpret_cast<size_t>(codes) & 15) == 0, "acmi_quantize_rows_i8: codes must be 16-byte aligned");
    QuantRowsArgs a = {x, dtype == ACMI_BF16, ldx, R, K, (K + 63) / 64, reinterpret_cast<uint8_t*>(codes), scale};
    hipLaunchKernelGGL(quant_rows_kernel, dim3(R), dim3(256), 0, (hipStream_t)stream, a);
    return acmi_check_launch("quant_rows_kernel");
}

// =====================================================================================================
// few rows: the weight is streamed once
// =====================================================================================================
// One workgroup per 16 output channels; its NW waves split K, every wave multiplies its weight fragments with MT 16-row blocks
// of the activation, and the integer partial sums meet in LDS (exact, so their order does not matter).  Transposed like the
// prefill GEMM: A operand = weight, so a lane ends with 4 consecutive channels of one row.
struct I8Args {
    const u32x4* a; const float* a_scale; const u32x4* w; const float* w_scale; const float* bias; const float* residual;
    void* out; int out_bf16; long long ldo; int act, M, N, K, nkc;
};

__device__ __forceinline__ void i8_mma(const u32x4& a, const u32x4& b, i32x4& acc) {
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), acc, 0, 0, 0);
}
__device__ __forceinline__ float i8_gelu(float x) { return 0.5f * x * (1.0f + erff(x * 0.70710678118654752440f)); }

template <int MT, int NW>
__global__ __launch_bounds__(NW * 64) void lin_i8_kernel(const I8Args p) {
    __shared__ i32x4 part[NW][MT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nt = blockIdx.x, mt0 = blockIdx.y * MT, mtiles = (p.M + 15) / 16;
    const u32x4* w = p.w + (size_t)nt * p.nkc * 64 + lane;
    i32x4 acc[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m] = i32x4{0, 0, 0, 0};
    for (int kc = wave; kc < p.nkc; kc += NW) {
        const u32x4 wf = __builtin_nontemporal_load(w + (size_t)kc * 64);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int mt = min(mt0 + m, mtiles - 1);
            const u32x4 af = p.a[((size_t)mt * p.nkc + kc) * 64 + lane];
            i8_mma(wf, af, acc[m]);
        }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) part[wave][m][lane] = acc[m];
    __syncthreads();
    for (int e = threadIdx.x; e < MT * 64; e += NW * 64) {
        const int m = e >> 6, ln = e & 63, row = (mt0 + m) * 16 + (ln & 15), col = nt * 16 + (ln >> 4) * 4;
        if (row >= p.M) continue;
        i32x4 s = part[0][m][ln];
#pragma unroll
        for (int k = 1; k < NW; ++k) s += part[k][m][ln];
        const float sa = p.a_scale[row];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int c = col + r;
            if (c >= p.N) break;
            float y = fmaf((float)s[r], sa * p.w_scale[c], p.bias != nullptr ? p.bias[c] : 0.f);
            if (p.act == 1) y = i8_gelu(y);
            if (p.residual != nullptr) y += p.residual[(size_t)row * p.N + c];
            const size_t at = (size_t)(row * p.ldo) + c;
            if (p.out_bf16) reinterpret_cast<bf16_t*>(p.out)[at] = f32_to_bf16(y);
            else reinterpret_cast<float*>(p.out)[at] = y;
        }
    }
}

extern "C" int acmi_linear_i8(const acmi_linear_i8_desc* desc, void* stream) {
    ACMI_REQUIRE(desc != nullptr, "acmi_linear_i8: null descriptor");
    const acmi_linear_i8_desc& d = *desc;
    ACMI_REQUIRE(d.M >= 0 && d.N > 0 && d.K > 0 && d.K <= 131072, "acmi_linear_i8: M=%d N=%d K=%d (K in [1, 131072])", d.M, d.N, d.K);
    ACMI_REQUIRE(d.out_dtype == ACMI_F32 || d.out_dtype == ACMI_BF16, "acmi_linear_i8: out_dtype %d", d.out_dtype);
    ACMI_REQUIRE(d.act == 0 || d.act == 1, "acmi_linear_i8: act %d", d.act);
    if (d.M == 0) return ACMI_OK;
    ACMI_REQUIRE(d.a && d.a_scale && d.w && d.w_scale && d.out && d.ldo >= d.N, "acmi_linear_i8: null operand or ldo=%lld < N=%d", d.ldo, d.N);
    ACMI_REQUIRE(((reinterpret_cast<size_t>(d.a) | reinterpret_cast<size_t>(d.w)) & 15) == 0, "acmi_linear_i8: codes must be 16-byte aligned");
    I8Args a = {};
    a.a = reinterpret_cast<const u32x4*>(d.a); a.a_scale = d.a_scale; a.w = reinterpret_cast<const u32x4*>(d.w); a.w_scale = d.w_scale;
    a.bias = d.bias; a.residual = d.residual; a.out = d.out; a.out_bf16 = d.out_dtype == ACMI_BF16; a.ldo = d.ldo;
    a.act = d.act; a.M = d.M; a.N = d.N; a.K = d.K; a.nkc = (d.K + 63) / 64;
    const int nt = (d.N + 15) / 16, mt = (d.M + 15) / 16;
    hipStream_t st = (hipStream_t)stream;
    if (d.M > 64) {
        BigArgs b = {};
        b.a = d.a; b.w = d.w; b.bias = d.bias; b.M = mt * 16; b.N = d.N; b.K = d.K; b.epi = ACMI_BIG_I8; b.act = d.act;
        b.a_scale = d.a_scale; b.w_scale = d.w_scale; b.residual = d.residual; b.rows = d.M;
        b.out = reinterpret_cast<float*>(d.out); b.out_bf16 = a.out_bf16; b.ldo64 = d.ldo;
        return acmi_launch_big_i8(b, st);
    }
    if (mt == 1) hipLaunchKernelGGL((lin_i8_kernel<1, 8>), dim3(nt, 1), dim3(512), 0, st, a);
    else if (mt == 2) hipLaunchKernelGGL((lin_i8_kernel<2, 8>), dim3(nt, 1), dim3(512), 0, st, a);
    else hipLaunchKernelGGL((lin_i8_kernel<4, 8>), dim3(nt, 1), dim3(512), 0, st, a);
    return acmi_check_launch("lin_i8_kernel");
}
