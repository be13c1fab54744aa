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
  int wide;                   // out is float32, else bfloat16
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

// ---------------------------------------------------------------- few rows
// A workgroup owns 16 NT rows of the weights (with GLU 8 NT gates and their ups) and all rows of x; its waves deal k out among
// them in chunks of 128 S and their sums meet in LDS in wave order. A load of the weights brings whole lines, eight blocks of
// eight rows; the matrix instruction wants four blocks of sixteen, so the halves of every sixteen lanes trade places between the
// loads of rows 0 to 7 and 8 to 15 (a move across lanes for each register, no LDS). x goes
// through a piece of LDS of the wave's own (no barrier) in whole lines: read as operands from memory each of its rows would
// cost a cache line an instruction and lane. The 16-byte pieces of a row are permuted by the row's number on the way in, so
// that the operand reads spread over the banks. R rows are brought whatever M is (the last one again), so that a chunk is a
// number of loads known when the code is compiled and the wait for one leaves the next on its way. What is left of k
// behind the whole chunks is one wave's, with loads that ask where k ends.
//
// Waves: every CU wants some 16 of them with two chunks each on their way, which 64 KB of weights in flight keep the memory
// busy with; fewer than four a workgroup leave too many of the sums' exchanges.
template <bool X8, bool GLU, int MT, int NT, int S, int R>
__global__ __launch_bounds__(MT > 1 ? 512 : 1024) void mx_few_kernel(MxGemm g, int bytes) {
  static_assert(!GLU || NT % 2 == 0, "gates and ups");
  static_assert(R <= 16 * MT && (S == 2 || S == 4), "rows of the tiles, loads in pairs");
  constexpr int P = (X8 ? 8 : 16) * S;          // 16-byte pieces of a row of x in a chunk
  constexpr int FLIP = P < 16 ? P - 1 : 15;
  constexpr int NO = GLU ? NT / 2 : NT;         // tiles of results
  constexpr int XI = R * P > 64 ? R * P / 64 : 1;               // loads of x
  constexpr int LOADS = XI + NT * (S + 1) + (X8 ? MT : 0);      // of a chunk: at least so many
  extern __shared__ __attribute__((aligned(16))) unsigned char mx_lds[];
  // (what is the same in a whole wave is told to be: addresses are then one base and 32 bits a lane)
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, r = lane % 16, q = lane / 16,
            waves = blockDim.x / 64;
  const int n0 = blockIdx.x * 16 * NO, blocks = g.K / MX_BLOCK, chunks = blocks / (4 * S);
  unsigned char* mine = mx_lds + wave * bytes;
  const uint8_t *codes[GLU ? 2 : 1], *scales[GLU ? 2 : 1];      // of the workgroup's first row, of its first ups
#pragma unroll
  for (int u = 0; u < (GLU ? 2 : 1); ++u) {
    codes[u] = g.codes + ((size_t)n0 + (u ? (size_t)g.N : 0)) * (g.K / 2);
    scales[u] = g.scales + ((size_t)n0 + (u ? (size_t)g.N : 0)) * blocks;
  }
  uint32_t col[NO];                             // this lane's row of the weights, from n0 on
#pragma unroll
  for (int t = 0; t < NO; ++t) col[t] = n0 + 16 * t + r < g.N ? 16 * t + r : g.N - 1 - n0;
  uint32_t piece_at[NO][2];                     // what this lane loads: a block of row r % 8, of row 8 + r % 8
#pragma unroll
  for (int t = 0; t < NO; ++t)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = 16 * t + 8 * h + r % 8;
      piece_at[t][h] = (uint32_t)(n0 + at < g.N ? at : g.N - 1 - n0) * (uint32_t)(g.K / 2) + (q + 4 * (r / 8)) * 16;
    }
  uint32_t row[MT];                             // and of x
#pragma unroll
  for (int m = 0; m < MT; ++m) row[m] = 16 * m + r < g.M ? 16 * m + r : g.M - 1;
  const uint32_t xstep = (uint32_t)g.ldx * (X8 ? 1 : 2);
  mx_f32x4 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[m][t] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
  mx_u32x4 w[2][NT][S];
  uint32_t ws[2][NT][S], xs[2][X8 ? MT : 1][S];

  // all that chunk c needs, x first: it comes from a cache, and a wait that is too long by a few loads waits for it
  const auto ask = [&](int set, int c) {
    unsigned char* to = mine + (size_t)set * R * P * 16;
#pragma unroll
    for (int i = 0; i < XI; ++i) {
      const uint32_t at = i * 64 + lane, lrow = at / P, from = (int)lrow < g.M ? lrow : g.M - 1;
      const uint32_t piece = (at % P) ^ (lrow & FLIP);
      if (R * P >= 64 || at < R * P)
        ta_load_to_lds16((const unsigned char*)g.x + (size_t)c * P * 16, from * xstep + piece * 16, to + i * 1024);
    }
    if (X8)
#pragma unroll
      for (int m = 0; m < MT; ++m) __builtin_memcpy(xs[set][m], g.xs + (size_t)c * 4 * S + row[m] * (uint32_t)blocks, 4 * S);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      __builtin_memcpy(ws[set][t], scales[t / NO] + (size_t)c * 4 * S + col[t % NO] * (uint32_t)blocks, 4 * S);
#pragma unroll
      for (int s = 0; s < S; ++s)
        w[set][t][s] = __builtin_nontemporal_load(
            reinterpret_cast<const mx_u32x4*>(codes[t / NO] + (size_t)(c * S + s / 2 * 2) * 64 + piece_at[t % NO][s % 2]));
    }
  };
  // loads 2 i and 2 i + 1 to operands of steps 2 i and 2 i + 1: lanes 8 to 15 of the first take the second's of lanes 0 to 7,
  // and the other way round
  const auto trade = [&](int set) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int s = 0; s < S; s += 2)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int a = (int)w[set][t][s][i], b = (int)w[set][t][s + 1][i];
          w[set][t][s][i] = (uint32_t)__builtin_amdgcn_update_dpp(a, b, 0x128, 0xf, 0xc, false);       // rotated by 8 in 16
          w[set][t][s + 1][i] = (uint32_t)__builtin_amdgcn_update_dpp(b, a, 0x128, 0xf, 0x3, false);
        }
  };
  const auto multiply = [&](int set) {
    const unsigned char* xl = mine + (size_t)set * R * P * 16;
    const auto piece = [&](int m, int p) {
      return *reinterpret_cast<const mx_u32x4*>(xl + ((size_t)row[m] * P + (p ^ (row[m] & FLIP))) * 16);
    };
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (X8) {
        // lane group q holds the halves q % 2 of the 128 k's blocks q / 2 and 2 + q / 2, and block q's scale
        mx_i32x8 a[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const mx_u32x4 lo = piece(m, 8 * s + q), hi = piece(m, 8 * s + 4 + q);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            a[m][i] = (int)lo[i];
            a[m][4 + i] = (int)hi[i];
          }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const mx_u32x4 c = w[set][t][s];
          const mx_i32x8 b = {(int)c[0], (int)c[1], (int)c[2], (int)c[3], 0, 0, 0, 0};
#pragma unroll
          for (int m = 0; m < MT; ++m)
            acc[m][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a[m], b, acc[m][t], 0, 4, 0, (int)(xs[set][m][s] >> (8 * q)), 0,
                                                                         (int)(ws[set][t][s] >> (8 * q)));
        }
      } else {
        union {
          mx_u32x4 u;
          mx_bf16x8 v;
        } a[MT][4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int j = 0; j < 4; ++j) a[m][j].u = piece(m, 16 * s + 4 * q + j);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float scale = mx_scale(ws[set][t][s] >> (8 * q) & 255u);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const mx_bf16x8 b = mx_widen8(w[set][t][s][j], scale);
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[m][j].v, b, acc[m][t], 0, 0, 0);
          }
        }
      }
    }
  };

  int c = wave;
  if (c < chunks) {
    ask(0, c);
    if (c + waves < chunks) ask(1, c + waves);
  }
  while (c < chunks) {
#pragma unroll
    for (int set = 0; set < 2; ++set) {
      if (c >= chunks) break;
      if (c + waves < chunks) ta_wait_loads<LOADS>();
      else ta_wait_loads<0>();
      __builtin_amdgcn_sched_barrier(0);
      trade(set);
      multiply(set);
      // the next load to this set's LDS goes out when its rows have been read
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      if (c + 2 * waves < chunks) ask(set, c + 2 * waves);
      __builtin_amdgcn_sched_barrier(0);
      c += waves;
    }
  }
  // blocks behind the last whole chunk: dead ones are zero in x and have the scale 1
  const int first = chunks * 4 * S;
  if (first < blocks && wave == chunks % waves) {
    const uint32_t pieces = g.K / (X8 ? 16 : 8);
#pragma unroll
    for (int i = 0; i < XI; ++i) {
      const uint32_t at = i * 64 + lane, lrow = at / P, from = (int)lrow < g.M ? lrow : g.M - 1;
      const uint32_t piece = chunks * P + ((at % P) ^ (lrow & FLIP));
      if (at < R * P) {
        mx_u32x4 v = {0, 0, 0, 0};
        if (piece < pieces)
          v = *reinterpret_cast<const mx_u32x4*>((const unsigned char*)g.x + from * xstep + (size_t)piece * 16);
        reinterpret_cast<mx_u32x4*>(mine)[at] = v;
      }
    }
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int b = first + 4 * s + q;
      const bool live = b < blocks;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        w[0][t][s] = mx_u32x4{0, 0, 0, 0};
        ws[0][t][s] = 0x7f7f7f7fu;
        if (live) {
          w[0][t][s] = *reinterpret_cast<const mx_u32x4*>(codes[t / NO] + (size_t)b * 16 + col[t % NO] * (uint32_t)(g.K / 2));
          ws[0][t][s] = (uint32_t)scales[t / NO][b + col[t % NO] * (uint32_t)blocks] * 0x01010101u;
        }
      }
      if (X8)
#pragma unroll
        for (int m = 0; m < MT; ++m) xs[0][m][s] = live ? (uint32_t)g.xs[b + row[m] * (uint32_t)blocks] * 0x01010101u : 0x7f7f7f7fu;
    }
    multiply(0);
  }
  // the sums, in the place of the wave's x
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  float* part = reinterpret_cast<float*>(mine);
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[(m * NT + t) * 256 + (q * 4 + i) * 16 + r] = acc[m][t][i];
  __syncthreads();
  for (int o = threadIdx.x; o < MT * NO * 256; o += blockDim.x) {
    const int mt = o / (NO * 256), t = o / 256 % NO, at = o % 256;
    const int m = 16 * mt + at / 16, n = n0 + 16 * t + at % 16;
    if (m >= g.M || n >= g.N) continue;
    float v[2] = {0.f, 0.f};
#pragma unroll
    for (int u = 0; u < (GLU ? 2 : 1); ++u) {
      const int tile = (mt * NT + t + u * NO) * 256 + at;
      for (int wv = 0; wv < waves; ++wv) v[u] += reinterpret_cast<const float*>(mx_lds + wv * bytes)[tile];
      if (g.bias) v[u] += g.bias[n + (long long)u * g.N];
    }
    const float y = GLU ? v[0] / (1.0f + expf(-v[0])) * v[1] : v[0];
    const long long to = (long long)m * g.ldo + n;
    if (g.wide) reinterpret_cast<float*>(g.out)[to] = y;
    else reinterpret_cast<bf16_t*>(g.out)[to] = from_f32<bf16_t>(y);
  }
}

#define MX_LDS (160 * 1024)
template <bool X8, bool GLU, int MT, int NT, int S, int R>
static int mx_few_launch(const char* what, hipStream_t stream, const MxGemm& g) {
  constexpr int P = (X8 ? 8 : 16) * S, MOST = MT > 1 ? 8 : 16, NO = GLU ? NT / 2 : NT;
  constexpr int x = R * P * 16, sums = MT * NT * 1024;
  const auto kernel = mx_few_kernel<X8, GLU, MT, NT, S, R>;
  const int chunks = g.K / (128 * S), grid = (g.N + NO * 16 - 1) / (NO * 16);
  // as many waves as give every CU 16, then the fewest that need as many turns; one buffer of x does for one turn
  int waves = (16 * 256 + grid - 1) / grid;
  waves = waves < 4 ? 4 : waves > MOST ? MOST : waves;
  if (waves > chunks) waves = chunks > 0 ? chunks : 1;
  int bytes = waves < chunks ? 2 * x : x;
  if (bytes < sums) bytes = sums;
  if (waves * bytes > MX_LDS) {
    bytes = 2 * x > sums ? 2 * x : sums;
    waves = MX_LDS / bytes;
  }
  const int turns = (chunks + waves - 1) / waves;
  if (turns > 0) waves = (chunks + turns - 1) / turns;
  static int allowed = 64 * 1024;
  if (waves * bytes > allowed) {
    const hipError_t e =
        hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, MX_LDS);
    if (e != hipSuccess) return ta_fail("%s: %d bytes of LDS refused (%s)", what, MX_LDS, hipGetErrorString(e));
    allowed = MX_LDS;
  }
  kernel<<<grid, waves * 64, (size_t)waves * bytes, stream>>>(g, bytes);
  return ta_check_launch(what);
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
  const MxGemm g = {x, nullptr, (const uint8_t*)codes, (const uint8_t*)scales, bias, out, ldx, ldo, M, N, K, out_dtype == TA_F32};
  if (mx_gemm_check("ta_gemm_mx4", g)) return 1;
  TA_REQUIRE(M <= MX_FEW_ROWS, "ta_gemm_mx4: %d bfloat16 rows, at most %d", M, MX_FEW_ROWS);
  TA_REQUIRE(ldx >= K && ldx % 8 == 0, "ta_gemm_mx4: rows %lld apart do not start on 16 bytes", ldx);
  TA_REQUIRE(ldx <= 1 << 24 && K <= 1 << 24, "ta_gemm_mx4: rows %lld apart, k %d: at most 16,777,216", ldx, K);   // 64 rows within 31 bits
  TA_REQUIRE(!swiglu || N <= 0x3fffffff, "ta_gemm_mx4: %d gates", N);
  if (M == 0) return 0;
  if (swiglu) {
    if (M <= 1) return mx_few_launch<false, true, 1, 2, 2, 1>("ta_gemm_mx4", stream, g);
    if (M <= 4) return mx_few_launch<false, true, 1, 2, 2, 4>("ta_gemm_mx4", stream, g);
    if (M <= 8) return mx_few_launch<false, true, 1, 2, 2, 8>("ta_gemm_mx4", stream, g);
    if (M <= 16) return mx_few_launch<false, true, 1, 2, 2, 16>("ta_gemm_mx4", stream, g);
    if (M <= 32) return mx_few_launch<false, true, 2, 2, 2, 32>("ta_gemm_mx4", stream, g);
    return mx_few_launch<false, true, 4, 2, 2, 64>("ta_gemm_mx4", stream, g);
  }
  if (M <= 1) return mx_few_launch<false, false, 1, 1, 4, 1>("ta_gemm_mx4", stream, g);
  if (M <= 4) return mx_few_launch<false, false, 1, 1, 4, 4>("ta_gemm_mx4", stream, g);
  if (M <= 8) return mx_few_launch<false, false, 1, 1, 4, 8>("ta_gemm_mx4", stream, g);
  if (M <= 16) return mx_few_launch<false, false, 1, 1, 2, 16>("ta_gemm_mx4", stream, g);
  if (M <= 32) return mx_few_launch<false, false, 2, 2, 2, 32>("ta_gemm_mx4", stream, g);
  return mx_few_launch<false, false, 4, 2, 2, 64>("ta_gemm_mx4", stream, g);
}

// 8-bit rows, codes [M][K] and bytes [M][K/32]; out bfloat16.
extern "C" int ta_gemm_mx4_mx8(hipStream_t stream, const void* x, const void* xs, const void* codes, const void* scales, const float* bias,
                               void* out, long long ldo, int M, int N, int K) {
  const MxGemm g = {x, (const uint8_t*)xs, (const uint8_t*)codes, (const uint8_t*)scales, bias, out, K, ldo, M, N, K, 0};
  if (mx_gemm_check("ta_gemm_mx4_mx8", g)) return 1;
  TA_REQUIRE(K <= 1 << 24, "ta_gemm_mx4_mx8: k %d: at most 16,777,216", K);
  if (M == 0) return 0;
  if (M <= 1) return mx_few_launch<true, false, 1, 1, 4, 1>("ta_gemm_mx4_mx8", stream, g);
  if (M <= 4) return mx_few_launch<true, false, 1, 1, 4, 4>("ta_gemm_mx4_mx8", stream, g);
  if (M <= 8) return mx_few_launch<true, false, 1, 1, 4, 8>("ta_gemm_mx4_mx8", stream, g);
  if (M <= 16) return mx_few_launch<true, false, 1, 1, 4, 16>("ta_gemm_mx4_mx8", stream, g);
  if (M <= 32) return mx_few_launch<true, false, 2, 2, 2, 32>("ta_gemm_mx4_mx8", stream, g);
  if (M <= 64) return mx_few_launch<true, false, 4, 2, 2, 64>("ta_gemm_mx4_mx8", stream, g);
  const int nt = (N + 15) / 16, grid = nt * ((M + 15) / 16);
  mx_gemm_kernel<true, false, bf16_t><<<grid, 256, 0, stream>>>(g, nt);
  return ta_check_launch("ta_gemm_mx4_mx8");
}
