// Projection in 8-bit integers, gfx950 (CDNA4, wave64): rows quantised with a scale each (tokens of an activation, output
// channels of a weight), int8 x int8 products summed exactly in 32-bit integers by the matrix cores, one f32 scaling at the end.
// Format: include/acmi.h.  Reference semantics: the nn.Linear projections of audiocraft/modules/transformer.py:362-399, 454-574.
#include "acmi_lm_internal.h"

#include <math.h>

typedef int i32x4 __attribute__((ext_vector_type(4)));

// =====================================================================================================
// rows -> int8 fragments + a scale each
// =====================================================================================================
struct RowSrc { const void* x; long long ldx; int bf16, R, K; };
// 4 elements of a row that starts anywhere: global loads need no more than the element's alignment (loaded one by one where a row
// does not start on 4 elements: 9187 x 4065 bf16 67 us, now 32; 9600 x 1535 21 and 14, as aligned ones)
typedef uint32_t row_u32x2 __attribute__((ext_vector_type(2), aligned(2)));
typedef float row_f32x4 __attribute__((ext_vector_type(4), aligned(4)));

// columns [col, col + 4) of a row; 0 past K
__device__ __forceinline__ f32x4 row_ld4(const RowSrc& s, size_t base, int col) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (col + 4 <= s.K) {
        if (s.bf16) {
            const row_u32x2 w = *reinterpret_cast<const row_u32x2*>(reinterpret_cast<const bf16_t*>(s.x) + base + col);
            v = f32x4{__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u), __uint_as_float(w[1] << 16), __uint_as_float(w[1] & 0xffff0000u)};
        } else {
            v = *reinterpret_cast<const row_f32x4*>(reinterpret_cast<const float*>(s.x) + base + col);
        }
        return v;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (col + e < s.K) v[e] = s.bf16 ? bf16_to_f32(reinterpret_cast<const bf16_t*>(s.x)[base + col + e]) : reinterpret_cast<const float*>(s.x)[base + col + e];
    return v;
}
__device__ __forceinline__ float row_max4(const f32x4& v, float m) {   // +infinity for a NaN, which fmaxf would drop
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float a = fabsf(v[e]);
        m = fmaxf(m, a <= 3.4028234663852886e38f ? a : INFINITY);
    }
    return m;
}
__device__ __forceinline__ void row_scale(float amax, float& scale, float& inv) {
    if (amax == INFINITY) { scale = __uint_as_float(0x7fc00000u); inv = 0.f; }
    else if (amax < 7.52316384526264e-37f) { scale = 0.f; inv = 0.f; }   // 2^-120: 127 / amax stays finite above
    else { scale = __fdiv_rn(amax, 127.f); inv = __fdiv_rn(127.f, amax); }
}
// 4 codes: the product rounded to f32, then to the nearest integer by adding 1.5 * 2^23 (ties to even, |product| <= 127 (1 +
// 2^-23)), whose low byte it then is.  (A row with a NaN has inv = 0; a NaN product gives some byte, its scale is NaN.)
__device__ __forceinline__ uint32_t row_codes4(const f32x4& v, float inv) {
    uint32_t b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = __float_as_uint(v[e] * inv + 12582912.f);
    const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
    return lo | hi;
}

struct QuantRowsArgs { RowSrc s; int nkc, kchunk; uint8_t* codes; float* scale; };

// One workgroup per 16 rows, a wave per row: the row is read once (NV x 256 columns of it stay in registers, longer ones are read
// again from L2), its codes are laid down in LDS, and the 16 rows leave as whole fragments, 1 KB at a time.  (One workgroup per row
// wrote 16-byte pieces 256 bytes apart: 38 us for 9600 x 1536 f32, now 13.2: 74 MB at 5.6 TB/s, part of it out of the last-level
// cache.)  9600 x 6144 f32, of whose rows a third is read twice: 65 us.
template <int NV>
__global__ __launch_bounds__(1024) void quant_rows_kernel(const QuantRowsArgs p) {
    extern __shared__ __attribute__((aligned(16))) unsigned char sm[];   // [16][kchunk + 16]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = blockIdx.x * 16 + wave, kpad = p.nkc * 64, pitch = p.kchunk + 16;
    const bool live = row < p.s.R;
    const size_t base = (size_t)((live ? row : 0) * p.s.ldx);
    f32x4 v[NV];
    float amax = 0.f;
    if (live) {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = row_ld4(p.s, base, (i * 64 + lane) * 4);
#pragma unroll
        for (int i = 0; i < NV; ++i) amax = row_max4(v[i], amax);
        for (int c = (NV * 64 + lane) * 4; c < p.s.K; c += 256) amax = row_max4(row_ld4(p.s, base, c), amax);
    }
    amax = wave_max(amax);
    float scale, inv;
    row_scale(amax, scale, inv);
    if (live && lane == 0) p.scale[row] = scale;
    for (int k0 = 0; k0 < kpad; k0 += p.kchunk) {   // (one round unless K > 8192)
        const int k1 = min(kpad, k0 + p.kchunk);
        if (k0 > 0) __syncthreads();
        uint32_t* dst = reinterpret_cast<uint32_t*>(sm + wave * pitch);
        if (!live) {
            for (int c = k0 + lane * 4; c < k1; c += 256) dst[(c - k0) >> 2] = 0;
        } else if (k0 == 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * 64 + lane) * 4;
                if (c < k1) dst[c >> 2] = row_codes4(v[i], inv);
            }
            for (int c = (NV * 64 + lane) * 4; c < k1; c += 256) dst[c >> 2] = row_codes4(row_ld4(p.s, base, c), inv);
        } else {
            for (int c = k0 + lane * 4; c < k1; c += 256) dst[(c - k0) >> 2] = row_codes4(row_ld4(p.s, base, c), inv);
        }
        __syncthreads();
        u32x4* out = reinterpret_cast<u32x4*>(p.codes) + ((size_t)blockIdx.x * p.nkc + (k0 >> 6)) * 64 + lane;
        for (int kc = wave; kc < (k1 - k0) >> 6; kc += 16)
            out[(size_t)kc * 64] = *reinterpret_cast<const u32x4*>(sm + (lane & 15) * pitch + kc * 64 + (lane >> 4) * 16);
    }
}

// few rows: one workgroup of 8 waves per row, all of it in flight at once (8192 columns in registers); the 16-byte pieces it writes
// lie 256 bytes apart, which costs nothing while there are few.  16 x 6144 f32: 9.5 -> 3.2 us
__global__ __launch_bounds__(512) void quant_row_wide_kernel(const QuantRowsArgs p) {
    constexpr int NV = 4, STEP = 512 * 4;
    __shared__ float red[8];
    extern __shared__ __attribute__((aligned(16))) unsigned char sm[];   // [kchunk]
    const int row = blockIdx.x, kpad = p.nkc * 64;
    const size_t base = (size_t)(row * p.s.ldx);
    f32x4 v[NV];
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = row_ld4(p.s, base, i * STEP + threadIdx.x * 4);
#pragma unroll
    for (int i = 0; i < NV; ++i) amax = row_max4(v[i], amax);
    for (int c = NV * STEP + threadIdx.x * 4; c < p.s.K; c += STEP) amax = row_max4(row_ld4(p.s, base, c), amax);
    amax = wave_max(amax);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = amax;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 8; ++k) amax = fmaxf(amax, red[k]);
    float scale, inv;
    row_scale(amax, scale, inv);
    if (threadIdx.x == 0) p.scale[row] = scale;
    uint32_t* dst = reinterpret_cast<uint32_t*>(sm);
    for (int k0 = 0; k0 < kpad; k0 += p.kchunk) {   // (one round unless K > 8192)
        const int k1 = min(kpad, k0 + p.kchunk);
        if (k0 > 0) __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = i * STEP + threadIdx.x * 4;
            if (k0 == 0) { if (c < k1) dst[c >> 2] = row_codes4(v[i], inv); }
            else if (k0 + c < k1) dst[c >> 2] = row_codes4(row_ld4(p.s, base, k0 + c), inv);
        }
        __syncthreads();
        for (int ch = threadIdx.x; ch < (k1 - k0) >> 4; ch += 512) {
            const int g = (k0 >> 4) + ch;   // chunk of 16 columns = 16 bytes of one lane of fragment g / 4
            const size_t frag = (size_t)(row >> 4) * p.nkc + (g >> 2);
            *reinterpret_cast<u32x4*>(p.codes + frag * 1024 + ((g & 3) * 16 + (row & 15)) * 16) = *reinterpret_cast<const u32x4*>(sm + ch * 16);
        }
    }
}

static RowSrc row_src(const void* x, int dtype, long long ldx, int R, int K) {
    return RowSrc{x, ldx, dtype == ACMI_BF16, R, K};
}
// rows of one launch: its work items, 64 a row, are counted in 32 bits (more are dropped without an error)
constexpr int QUANT_MAX_ROWS = 1 << 25;
static int launch_quant_rows(const RowSrc& s, uint8_t* codes, float* scale, hipStream_t st) {
    QuantRowsArgs a = {s, (s.K + 63) / 64, 0, codes, scale};
    a.kchunk = min(a.nkc * 64, 8192);
    // A workgroup per row until they are many; then 16 rows to one, whose wave keeps 2048 columns of its row, 4096 where K is more, and
    // reads the rest again: those change over later.  us in a graph, per row / 16 rows: 384 x 1536 f32 4.2 / 4.6, 1000 x 1000 5.7 / 4.9,
    // 2048 x 2048 9.8 / 5.6, 4096 x 1536 15.1 / 5.9; 1024 x 4096 8.0 / 8.9, 2048 x 4096 12.8 / 10.5, 1024 x 6144 9.5 / 11.5, 2048 x 6144
    // 17.3 / 16.4 (bf16 15.3 / 17.4), 4096 x 6144 32.4 / 24.1, 2048 x 8000 bf16 19.5 / 23.2
    if (s.R <= (s.K > 2048 ? 2048 : 512)) {
        hipLaunchKernelGGL(quant_row_wide_kernel, dim3(s.R), dim3(512), (size_t)a.kchunk, st, a);
        return acmi_check_launch("quant_row_wide_kernel");
    }
    const size_t lds = (size_t)16 * (a.kchunk + 16);
    static const bool ok = hipFuncSetAttribute(reinterpret_cast<const void*>(&quant_rows_kernel<8>), hipFuncAttributeMaxDynamicSharedMemorySize, 16 * (8192 + 16)) == hipSuccess &&
                           hipFuncSetAttribute(reinterpret_cast<const void*>(&quant_rows_kernel<2>), hipFuncAttributeMaxDynamicSharedMemorySize, 16 * (8192 + 16)) == hipSuccess &&
                           hipFuncSetAttribute(reinterpret_cast<const void*>(&quant_rows_kernel<16>), hipFuncAttributeMaxDynamicSharedMemorySize, 16 * (8192 + 16)) == hipSuccess;
    ACMI_REQUIRE(ok, "acmi_quantize_rows_i8: cannot set the dynamic LDS limit");
    if (s.R > QUANT_MAX_ROWS) {
        for (int r0 = 0; r0 < s.R; r0 += QUANT_MAX_ROWS) {
            const int n = min(s.R - r0, QUANT_MAX_ROWS);
            const void* x = reinterpret_cast<const char*>(s.x) + (size_t)(r0 * s.ldx) * (s.bf16 ? 2 : 4);
            if (int rc = launch_quant_rows(RowSrc{x, s.ldx, s.bf16, n, s.K}, codes + (size_t)(r0 / 16) * a.nkc * 1024, scale + r0, st)) return rc;
        }
        return ACMI_OK;
    }
    if (s.K <= 512) hipLaunchKernelGGL(quant_rows_kernel<2>, dim3((s.R + 15) / 16), dim3(1024), lds, st, a);
    // (16 x 256 columns in registers halve the workgroups per CU; us 8 x 256 / 16 x 256: 9600 x 6144 f32 77 / 65, bf16 62 / 53, 4096 x 8000
    // bf16 31 / 28; 8192 x 4096 bf16 21.5 / 26, 9600 x 2100 16.3 / 25.9)
    else if (s.K > 4096) hipLaunchKernelGGL(quant_rows_kernel<16>, dim3((s.R + 15) / 16), dim3(1024), lds, st, a);
    else hipLaunchKernelGGL(quant_rows_kernel<8>, dim3((s.R + 15) / 16), dim3(1024), lds, st, a);
    return acmi_check_launch("quant_rows_kernel");
}

extern "C" int acmi_quantize_rows_i8(const void* x, int dtype, long long ldx, int R, int K, void* codes, float* scale, void* stream) {
    ACMI_REQUIRE(dtype == ACMI_F32 || dtype == ACMI_BF16, "acmi_quantize_rows_i8: dtype %d", dtype);
    ACMI_REQUIRE(R >= 0 && K > 0 && K <= 131072, "acmi_quantize_rows_i8: R=%d K=%d (K in [1, 131072])", R, K);
    if (R == 0) return ACMI_OK;
    ACMI_REQUIRE(R <= 1 << 30, "acmi_quantize_rows_i8: R=%d (at most 2^30)", R);
    ACMI_REQUIRE(x && codes && scale && ldx >= K, "acmi_quantize_rows_i8: null buffer or ldx=%lld < K=%d", ldx, K);
    ACMI_REQUIRE((reinterpret_cast<size_t>(codes) & 15) == 0, "acmi_quantize_rows_i8: codes must be 16-byte aligned");
    return launch_quant_rows(row_src(x, dtype, ldx, R, K), reinterpret_cast<uint8_t*>(codes), scale, (hipStream_t)stream);
}

// =====================================================================================================
// few rows: the weight is streamed once
// =====================================================================================================
// One workgroup per 16 output channels (and MT 16-row blocks); its NW waves split K, every wave multiplies its weight fragments
// with MT row blocks of the activation, and the integer partial sums meet in LDS (exact, so their order does not matter).
// Transposed like the prefill GEMM: A operand = weight, so a lane ends with 4 consecutive channels of one row.  The first WF
// weight fragments of a wave (and, for one row block, its activation's) are requested before anything else: up to K = 4096 with 8
// waves, 8192 with 16, a call is one round trip to memory.
// FUSED (at most 16 rows): the workgroup quantises the activation itself, into LDS, while its weights arrive -- a launch less.
struct I8Args {
    const u32x4* a; const float* a_scale; const u32x4* w; const float* w_scale; const float* bias; const float* residual;
    void* out; int out_bf16; long long ldo; int act, M, N, K, nkc;
    RowSrc s;
};
constexpr int I8_WF = 8;

__device__ __forceinline__ void i8_mma(const u32x4& a, const u32x4& b, i32x4& acc) {
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), acc, 0, 0, 0);
}
__device__ __forceinline__ float i8_gelu(float x) { return 0.5f * x * (1.0f + erff(x * 0.70710678118654752440f)); }

template <int MT, int NW, bool FUSED>
__global__ __launch_bounds__(NW * 64) void lin_i8_kernel(const I8Args p) {
    constexpr int WF = I8_WF, NV = 4;
    constexpr bool AF = MT == 1 && !FUSED;   // the activation's fragments are requested next to the weight's
    __shared__ i32x4 part[NW][MT][64];
    __shared__ float red[FUSED ? NW : 1], fscale[FUSED ? 16 : 1];
    extern __shared__ __attribute__((aligned(16))) unsigned char sm[];   // FUSED: [16][nkc * 64 + 16] codes
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nt = blockIdx.x, mt0 = blockIdx.y * MT, mtiles = (p.M + 15) / 16;
    const u32x4* w = p.w + (size_t)nt * p.nkc * 64 + lane;
    u32x4 wf[WF];
#pragma unroll
    for (int f = 0; f < WF; ++f) wf[f] = __builtin_nontemporal_load(w + (size_t)min(wave + f * NW, p.nkc - 1) * 64);
    u32x4 apre[AF ? WF : 1];
    if constexpr (AF) {
#pragma unroll
        for (int f = 0; f < WF; ++f) apre[f] = p.a[((size_t)min(mt0, mtiles - 1) * p.nkc + min(wave + f * NW, p.nkc - 1)) * 64 + lane];
        __builtin_amdgcn_sched_barrier(0);   // (the scheduler sinks the requests to their uses)
    }
    const int pitch = p.nkc * 64 + 16;
    if constexpr (FUSED) {
        // NW / M waves to a row (a power of two), rows in rounds of NW / wpr
        int wpr = 1;
        while (wpr * 2 * p.M <= NW) wpr *= 2;
        const int rpr = NW / wpr, mine = wave & (wpr - 1), step = wpr * 256;
        for (int r0 = 0; r0 < p.M; r0 += rpr) {
            const int row = r0 + wave / wpr;
            const bool live = row < p.M;
            const size_t base = (size_t)((live ? row : 0) * p.s.ldx);
            f32x4 v[NV];
            float amax = 0.f;
            if (live) {
#pragma unroll
                for (int i = 0; i < NV; ++i) v[i] = row_ld4(p.s, base, i * step + (mine * 64 + lane) * 4);
#pragma unroll
                for (int i = 0; i < NV; ++i) amax = row_max4(v[i], amax);
                for (int c = NV * step + (mine * 64 + lane) * 4; c < p.K; c += step) amax = row_max4(row_ld4(p.s, base, c), amax);
            }
            amax = wave_max(amax);
            if (wpr > 1) {   // (one round only)
                if (lane == 0) red[wave] = amax;
                __syncthreads();
                for (int k = 0; k < wpr; ++k) amax = fmaxf(amax, red[(wave & ~(wpr - 1)) + k]);
            }
            float scale, inv;
            row_scale(amax, scale, inv);
            if (live) {
                if (mine == 0 && lane == 0) fscale[row] = scale;
                uint32_t* dst = reinterpret_cast<uint32_t*>(sm + row * pitch);
                const int kpad = p.nkc * 64;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int c = i * step + (mine * 64 + lane) * 4;
                    if (c < kpad) dst[c >> 2] = row_codes4(v[i], inv);
                }
                for (int c = NV * step + (mine * 64 + lane) * 4; c < kpad; c += step) dst[c >> 2] = row_codes4(row_ld4(p.s, base, c), inv);
            }
        }
        __syncthreads();
    }
    i32x4 acc[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m] = i32x4{0, 0, 0, 0};
    auto mul = [&](int kc, const u32x4& wk) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            u32x4 af;   // (a row that does not exist only reaches outputs that are not stored)
            if constexpr (FUSED) af = *reinterpret_cast<const u32x4*>(sm + (lane & 15) * pitch + kc * 64 + (lane >> 4) * 16);
            else af = p.a[((size_t)min(mt0 + m, mtiles - 1) * p.nkc + kc) * 64 + lane];
            i8_mma(wk, af, acc[m]);
        }
    };
#pragma unroll
    for (int f = 0; f < WF; ++f)
        if (wave + f * NW < p.nkc) {
            if constexpr (AF) i8_mma(wf[f], apre[f], acc[0]);
            else mul(wave + f * NW, wf[f]);
        }
    for (int k0 = wave + WF * NW; k0 < p.nkc; k0 += WF * NW) {
#pragma unroll
        for (int f = 0; f < WF; ++f) wf[f] = __builtin_nontemporal_load(w + (size_t)min(k0 + f * NW, p.nkc - 1) * 64);
#pragma unroll
        for (int f = 0; f < WF; ++f)
            if (k0 + f * NW < p.nkc) mul(k0 + f * NW, wf[f]);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) part[wave][m][lane] = acc[m];
    __syncthreads();
    for (int e = threadIdx.x; e < MT * 256; e += NW * 64) {   // one output per thread
        const int m = e >> 8, n = e & 15, rl = (e >> 4) & 15, row = (mt0 + m) * 16 + rl, c = nt * 16 + n;
        if (row >= p.M || c >= p.N) continue;
        int sum = 0;
#pragma unroll
        for (int k = 0; k < NW; ++k) sum += reinterpret_cast<const int*>(&part[k][m][(n >> 2) * 16 + rl])[n & 3];
        const float sa = FUSED ? fscale[FUSED ? rl : 0] : p.a_scale[row];
        float y = fmaf((float)sum, sa * p.w_scale[c], p.bias != nullptr ? p.bias[c] : 0.f);
        if (p.act == 1) y = p.out_bf16 ? i8_gelu_bf16(y) : i8_gelu(y);
        if (p.residual != nullptr) y += p.residual[(size_t)row * p.N + c];
        const size_t at = (size_t)(row * p.ldo) + c;
        if (p.out_bf16) reinterpret_cast<bf16_t*>(p.out)[at] = f32_to_bf16(y);
        else reinterpret_cast<float*>(p.out)[at] = y;
    }
}

// Every workgroup of the fused form quantises the whole activation: while that is little.  Measured, us fused / two launches:
// 1 x 4096 x 1024 4.3 / 6.0, 8 x 1536 x 1536 4.8 / 7.0, 16 x 4096 x 1024 5.3 / 6.3; 16 x 4608 x 1536 8.0 / 7.2, 16 x 1536 x 6144 22 / 9.3
static bool i8_fused(int M, int K) { return M <= 16 && (long long)M * K <= 20480 && K <= 8192; }
static size_t i8_codes_bytes(int M, int K) { return (size_t)((M + 15) / 16) * ((K + 63) / 64) * 1024; }

extern "C" size_t acmi_linear_i8_work_bytes(int M, int K) {
    return M <= 0 || K <= 0 || i8_fused(M, K) ? 0 : i8_codes_bytes(M, K) + (size_t)M * sizeof(float);
}

extern "C" int acmi_linear_i8(const acmi_linear_i8_desc* desc, void* stream) {
    ACMI_REQUIRE(desc != nullptr, "acmi_linear_i8: null descriptor");
    const acmi_linear_i8_desc& d = *desc;
    ACMI_REQUIRE(d.M >= 0 && d.N > 0 && d.K > 0 && d.K <= 131072, "acmi_linear_i8: M=%d N=%d K=%d (K in [1, 131072])", d.M, d.N, d.K);
    ACMI_REQUIRE(d.out_dtype == ACMI_F32 || d.out_dtype == ACMI_BF16, "acmi_linear_i8: out_dtype %d", d.out_dtype);
    ACMI_REQUIRE(d.act == 0 || d.act == 1, "acmi_linear_i8: act %d", d.act);
    if (d.M == 0) return ACMI_OK;
    ACMI_REQUIRE(d.M <= 1 << 30 && d.N <= 1 << 30 && (long long)d.M * d.N <= 1LL << 38, "acmi_linear_i8: M=%d N=%d (each at most 2^30, M N at most 2^38)", d.M, d.N);
    ACMI_REQUIRE(d.N <= 1 << 25, "acmi_linear_i8: N=%d (at most 2^25: a launch counts its work items in 32 bits)", d.N);
    ACMI_REQUIRE(d.w && d.w_scale && d.out && d.ldo >= d.N, "acmi_linear_i8: null operand or ldo=%lld < N=%d", d.ldo, d.N);
    ACMI_REQUIRE((d.x != nullptr) != (d.a != nullptr && d.a_scale != nullptr), "acmi_linear_i8: either x or the quantised a, a_scale");
    ACMI_REQUIRE(((reinterpret_cast<size_t>(d.a) | reinterpret_cast<size_t>(d.w) | reinterpret_cast<size_t>(d.work)) & 15) == 0,
                 "acmi_linear_i8: codes and work must be 16-byte aligned");
    I8Args a = {};
    a.a = reinterpret_cast<const u32x4*>(d.a); a.a_scale = d.a_scale; a.w = reinterpret_cast<const u32x4*>(d.w); a.w_scale = d.w_scale;
    a.bias = d.bias; a.residual = d.residual; a.out = d.out; a.out_bf16 = d.out_dtype == ACMI_BF16; a.ldo = d.ldo;
    a.act = d.act; a.M = d.M; a.N = d.N; a.K = d.K; a.nkc = (d.K + 63) / 64;
    const int nt = (d.N + 15) / 16, mt = (d.M + 15) / 16;
    hipStream_t st = (hipStream_t)stream;
    if (d.x != nullptr) {
        ACMI_REQUIRE(d.x_dtype == ACMI_F32 || d.x_dtype == ACMI_BF16, "acmi_linear_i8: x_dtype %d", d.x_dtype);
        ACMI_REQUIRE(d.ldx >= d.K, "acmi_linear_i8: ldx=%lld < K=%d", d.ldx, d.K);
        a.s = row_src(d.x, d.x_dtype, d.ldx, d.M, d.K);
        if (i8_fused(d.M, d.K)) {
            static const bool ok = hipFuncSetAttribute(reinterpret_cast<const void*>(&lin_i8_kernel<1, 8, true>), hipFuncAttributeMaxDynamicSharedMemorySize, 16 * (8192 + 16)) == hipSuccess;
            ACMI_REQUIRE(ok, "acmi_linear_i8: cannot set the dynamic LDS limit");
            hipLaunchKernelGGL((lin_i8_kernel<1, 8, true>), dim3(nt, 1), dim3(512), (size_t)16 * (a.nkc * 64 + 16), st, a);
            return acmi_check_launch("lin_i8_kernel");
        }
        ACMI_REQUIRE(d.work != nullptr, "acmi_linear_i8: needs acmi_linear_i8_work_bytes bytes of work");
        uint8_t* codes = reinterpret_cast<uint8_t*>(d.work);
        float* scale = reinterpret_cast<float*>(codes + i8_codes_bytes(d.M, d.K));
        if (int rc = launch_quant_rows(a.s, codes, scale, st)) return rc;
        a.a = reinterpret_cast<const u32x4*>(codes); a.a_scale = scale;
    }
    // the tiled form once its 128 x 128 tiles give 3 of 8 CUs one; below, 64-row groups of the streaming form -- unless the
    // activation is larger than the L2s, from which the streaming form reads it once per 16 columns.  Measured without the
    // quantiser, us tiled / streamed: 256 x 4608 x 1536 (72 tiles) 12.3 / 12.0, 1000 x 1000 x 1000 (64) 10.5 / 9.0;
    // 1024 x 1536 x 6144 (96) 27.2 / 43.8, 512 x 4096 x 1024 (128) 10.5 / 15.9, 600 x 6144 x 1536 (240) 13.2 / 35.3; large
    // activations: 9187 x 117 x 4065 (72) 23.6 / 44.0, 9600 x 100 x 1536 (75) 11.9 / 21.8, 4800 x 100 x 3000 (38) 16.7 / 20.1, but
    // 2000 x 100 x 8000 (16) 31.6 / 21.5, 9600 x 30 x 4096 (75, of two column groups) 23.1 / 15.5
    const long long tiles = (long long)((d.M + 127) / 128) * ((d.N + 127) / 128);
    if (tiles >= 96 || (tiles >= 32 && d.N > 64 && (long long)d.M * d.K >= 1 << 23)) {
        BigArgs b = {};
        b.a = a.a; b.w = d.w; b.bias = d.bias; b.M = mt * 16; b.N = d.N; b.K = d.K; b.act = d.act;
        b.a_scale = a.a_scale; b.w_scale = d.w_scale; b.residual = d.residual; b.rows = d.M;
        b.out = reinterpret_cast<float*>(d.out); b.out_bf16 = a.out_bf16; b.ldo64 = d.ldo;
        return acmi_launch_big_i8(b, st);
    }
    if (mt == 1 && a.nkc > 64) hipLaunchKernelGGL((lin_i8_kernel<1, 16, false>), dim3(nt, 1), dim3(1024), 0, st, a);
    else if (mt == 1) hipLaunchKernelGGL((lin_i8_kernel<1, 8, false>), dim3(nt, 1), dim3(512), 0, st, a);
    else if (mt == 2) hipLaunchKernelGGL((lin_i8_kernel<2, 8, false>), dim3(nt, 1), dim3(512), 0, st, a);
    else hipLaunchKernelGGL((lin_i8_kernel<4, 8, false>), dim3(nt, (mt + 3) / 4), dim3(512), 0, st, a);
    return acmi_check_launch("lin_i8_kernel");
}
