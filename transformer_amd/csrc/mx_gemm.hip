// out[m, n] = sum over k of x[m, k] w[n, k] with 4-bit weights (mx.h), x in bfloat16 or in 8-bit blocks.
//
// bfloat16 rows: a power of two times an e2m1 value is a bfloat16, so the codes are widened exactly
// (v_cvt_scalef32_pk_bf16_fp4, two an instruction, scale included) and the products run on v_mfma_f32_16x16x32_bf16 with
// float32 sums.
//
// 8-bit rows: v_mfma_scale_f32_16x16x128_f8f6f4 takes both operands and both scales as they are. It lines up the 128 products
// of a call to the largest one's exponent before it adds them, which leaves some 15 bits below it (measured: 5e-5 of the sum
// of magnitudes where the operands' exponents fill their range); results are therefore bfloat16, which rounds 80 times as
// coarsely, and only the running sums over k are float32.
#include "mx.h"

__device__ __forceinline__ mx_bf16x8 mx_widen8(uint32_t codes, float scale) {
  union {
    mx_bf16x2 h[4];
    mx_bf16x8 v;
  } r;
  r.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
  r.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
  r.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
  r.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
  return r.v;
}

struct MxGemm {
  const void* x;              // bfloat16 [M][ldx], or e4m3 codes [M][K]
  const uint8_t* xs;          // bytes [M][K/32] of 8-bit rows
  const uint8_t* codes;       // [N][K/2], with gates N + N rows
  const uint8_t* scales;      // [N][K/32]
  const float* bias;          // per row of the weights, or null
  void* out;                  // [M][ldo]
  long long ldx, ldo;
  int M, N, K;
};

// One tile of 16 x 16 results a workgroup, whose four waves take every fourth 128 k; their sums meet in LDS in wave order.
// GLU: two tiles, gates and ups, joined before they are stored.
template <bool X8, bool GLU, typename TO>
__global__ __launch_bounds__(256) void mx_gemm_kernel(MxGemm g, int n_tiles) {
  constexpr int NT = GLU ? 2 : 1;
  __shared__ float part[4][NT][256];
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, r = lane % 16, q = lane / 16;
  const int n0 = (int)(blockIdx.x % n_tiles) * 16, m0 = (int)(blockIdx.x / n_tiles) * 16;
  const int blocks = g.K / MX_BLOCK;
  const long long m = m0 + r < g.M ? m0 + r : g.M - 1;
  const long long n = n0 + r < g.N ? n0 + r : g.N - 1;
  mx_f32x4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s = wave; s * 4 < blocks; s += 4) {
    const int b = s * 4 + q;                     // the block of this lane's weights
    const bool live = b < blocks;
    mx_u32x4 c[NT];
    uint32_t cs[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      c[t] = mx_u32x4{0, 0, 0, 0};
      cs[t] = 127;
      if (live) {
        const long long row = n + (long long)t * g.N;
        c[t] = *reinterpret_cast<const mx_u32x4*>(g.codes + row * (g.K / 2) + b * 16);
        cs[t] = g.scales[row * blocks + b];
      }
    }
    if (X8) {
      // lane group q holds the halves (q % 2) of the 128 k's blocks q / 2 and 2 + q / 2, and block q's scale
      const uint8_t* x = (const uint8_t*)g.x + m * g.K + s * 128;
      mx_i32x8 a = {0, 0, 0, 0, 0, 0, 0, 0};
      if (s * 4 + q / 2 < blocks) {
        const mx_u32x4 v = *reinterpret_cast<const mx_u32x4*>(x + q * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = (int)v[i];
      }
      if (s * 4 + 2 + q / 2 < blocks) {
        const mx_u32x4 v = *reinterpret_cast<const mx_u32x4*>(x + 64 + q * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) a[4 + i] = (int)v[i];
      }
      const int as = live ? g.xs[m * blocks + b] : 127;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const mx_i32x8 w = {(int)c[t][0], (int)c[t][1], (int)c[t][2], (int)c[t][3], 0, 0, 0, 0};
        acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, w, acc[t], 0, 4, 0, as, 0, (int)cs[t]);
      }
    } else {
      const bf16_t* x = (const bf16_t*)g.x + m * g.ldx + b * 32;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        union {
          mx_u32x4 u;
          mx_bf16x8 v;
        } a;
        a.u = mx_u32x4{0, 0, 0, 0};
        if (live) a.u = *reinterpret_cast<const mx_u32x4*>(x + j * 8);
#pragma unroll
        for (int t = 0; t < NT; ++t)
          acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, mx_widen8(c[t][j], mx_scale(cs[t])), acc[t], 0, 0, 0);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[wave][t][(q * 4 + i) * 16 + r] = acc[t][i];
  __syncthreads();
  const int mi = threadIdx.x / 16, ni = threadIdx.x % 16;
  if (m0 + mi >= g.M || n0 + ni >= g.N) return;
  float v[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    v[t] = part[0][t][threadIdx.x] + part[1][t][threadIdx.x] + part[2][t][threadIdx.x] + part[3][t][threadIdx.x];
    if (g.bias) v[t] += g.bias[n0 + ni + t * g.N];
  }
  const float y = GLU ? v[0] / (1.0f + expf(-v[0])) * v[NT - 1] : v[0];
  ((TO*)g.out)[(long long)(m0 + mi) * g.ldo + n0 + ni] = from_f32<TO>(y);
}

static int mx_gemm_check(const char* what, const MxGemm& g) {
  TA_REQUIRE(g.M >= 0 && g.N >= 1 && g.K >= MX_BLOCK && g.K % MX_BLOCK == 0, "%s: M=%d N=%d K=%d: k goes by blocks of %d", what, g.M, g.N, g.K,
             MX_BLOCK);
  TA_REQUIRE(g.ldo >= g.N, "%s: rows of %d results lie %lld apart", what, g.N, g.ldo);
  TA_REQUIRE((uintptr_t)g.x % 16 == 0 && (uintptr_t)g.codes % 16 == 0, "%s: operands do not start on 16 bytes", what);
  TA_REQUIRE((((long long)g.M + 15) / 16) * (((long long)g.N + 15) / 16) <= 0x7fffffffLL, "%s: M=%d N=%d are more than a launch holds", what,
             g.M, g.N);
  return 0;
}

// bfloat16 rows x [M][ldx] (rows on 16 bytes), at most ta_mx4_max_rows of them; out_dtype float32 or bfloat16; swiglu: the weights are N
// gate rows and N up rows.
#define MX_FEW_ROWS 64
extern "C" int ta_mx4_max_rows() { return MX_FEW_ROWS; }
extern "C" int ta_gemm_mx4(hipStream_t stream, int out_dtype, int swiglu, const void* x, long long ldx, const void* codes, const void* scales,
                           const float* bias, void* out, long long ldo, int M, int N, int K) {
  TA_REQUIRE(out_dtype == TA_F32 || out_dtype == TA_BF16, "ta_gemm_mx4: unknown dtype %d", out_dtype);
  const MxGemm g = {x, nullptr, (const uint8_t*)codes, (const uint8_t*)scales, bias, out, ldx, ldo, M, N, K};
  if (mx_gemm_check("ta_gemm_mx4", g)) return 1;
  TA_REQUIRE(M <= MX_FEW_ROWS, "ta_gemm_mx4: %d bfloat16 rows, at most %d", M, MX_FEW_ROWS);
  TA_REQUIRE(ldx >= K && ldx % 8 == 0, "ta_gemm_mx4: rows %lld apart do not start on 16 bytes", ldx);
  TA_REQUIRE(!swiglu || N <= 0x3fffffff, "ta_gemm_mx4: %d gates", N);
  if (M == 0) return 0;
  const int nt = (N + 15) / 16, grid = nt * ((M + 15) / 16);
  if (swiglu && out_dtype == TA_F32) mx_gemm_kernel<false, true, float><<<grid, 256, 0, stream>>>(g, nt);
  else if (swiglu) mx_gemm_kernel<false, true, bf16_t><<<grid, 256, 0, stream>>>(g, nt);
  else if (out_dtype == TA_F32) mx_gemm_kernel<false, false, float><<<grid, 256, 0, stream>>>(g, nt);
  else mx_gemm_kernel<false, false, bf16_t><<<grid, 256, 0, stream>>>(g, nt);
  return ta_check_launch("ta_gemm_mx4");
}

// 8-bit rows, codes [M][K] and bytes [M][K/32]; out bfloat16.
extern "C" int ta_gemm_mx4_mx8(hipStream_t stream, const void* x, const void* xs, const void* codes, const void* scales, const float* bias,
                               void* out, long long ldo, int M, int N, int K) {
  const MxGemm g = {x, (const uint8_t*)xs, (const uint8_t*)codes, (const uint8_t*)scales, bias, out, K, ldo, M, N, K};
  if (mx_gemm_check("ta_gemm_mx4_mx8", g)) return 1;
  if (M == 0) return 0;
  const int nt = (N + 15) / 16, grid = nt * ((M + 15) / 16);
  mx_gemm_kernel<true, false, bf16_t><<<grid, 256, 0, stream>>>(g, nt);
  return ta_check_launch("ta_gemm_mx4_mx8");
}
