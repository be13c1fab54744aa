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
#include <type_traits>
#include <stdlib.h>

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

// ---------------------------------------------------------------- many 8-bit rows
// Tiles of BM rows by BN columns, k by steps of 128 (one matrix instruction). Both operands come into LDS without registers in
// between, NS - 1 steps ahead, and so do the scales of every four steps (a row's are four bytes a step in a line of their own:
// step by step they cost as many requests as the operands).
//
// Eight waves, two on every SIMD, in two groups half a phase apart: while one group reads its operands from LDS the other
// multiplies, and a barrier ends the phase for both. KG 1: the groups are halves of the tile and take every step, in two phases;
// KG 2, for tiles that are too small to feed eight waves: each group has the whole tile and every second step, and the
// first adds the other's sums at the end. A phase waits until the loads that the next one reads are done, later ones stay under
// way; a place in LDS is loaded again once a barrier has passed since it was read. Towards the end of k there are fewer loads than
// a wait counts on, so the last phases wait for all of them.
//
// The weights are the first operand: a lane then holds 4 neighbouring columns of one row. Row p of the tile t of 16 stands for
// column 16 (p / 4) + 4 t + p % 4 of the wave's 64, so a lane's four tiles are 16 neighbouring columns, stored 16 bytes at a time.
// Pieces of 16 bytes are permuted by the row's number, so that eight lanes' reads meet no bank twice.
struct MxTiles {
  const uint8_t *xs, *ws;     // scales in rows of `step` bytes, a multiple of 16, 127 behind the last block
  int step;
  int m_tiles, n_tiles;
};

// 16 bytes a lane to the LDS that starts at `lds`; base and lds are the whole wave's
__device__ __forceinline__ void mx_to_lds16(const void* base, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(lds) : "m0", "memory");
}

template <int BM, int BN, int WM, int WN, int KG, int NS>
__global__ __launch_bounds__(512) void mx_tile_kernel(MxGemm g, MxTiles z) {
  constexpr int W = 8, TM = BM / (16 * WM);
  constexpr int XL = BM / 8 / W, WL = BN / 16 / W;             // loads of 1 KB a wave and step
  constexpr int SL = (BM + BN) / 64;                           // loads of 64 rows' scales, one a wave
  constexpr int LOADS = XL + WL;
  constexpr int AT_W = BM * 128, STAGE = AT_W + BN * 64, AT_S = NS * STAGE, GROUP = (BM + BN) * 16;
  static_assert(BN == 64 * WN && WM * WN * KG == W && BM % (16 * WM) == 0, "eight waves");
  static_assert(XL * 8 * W == BM && WL * 16 * W == BN && SL <= W && NS <= 4, "tiles in whole loads");
  extern __shared__ __attribute__((aligned(16))) unsigned char mx_lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, r = lane % 16, q = lane / 16;
  const int group = wave / 4, part = KG == 2 ? wave % 4 : wave, wm = part / WN, wn = part % WN;
  // workgroups go round the 8 XCDs: each gets neighbouring tiles, all rows of a band of columns, so that its cache holds them
  const int tiles = z.m_tiles * z.n_tiles, per = tiles / 8, b = blockIdx.x;
  const int tile = b < per * 8 ? (b % 8) * per + b / 8 : b;
  const int m0 = tile % z.m_tiles * BM, n0 = tile / z.m_tiles * BN;
  const int steps = (g.K + 127) / 128, pieces = g.K / 16, full = g.K / 128;
  const unsigned char* x = (const unsigned char*)g.x + (size_t)m0 * g.K;
  const unsigned char* w = g.codes + (size_t)n0 * (g.K / 2);

  uint32_t xo[XL], wo[WL], so;
#pragma unroll
  for (int i = 0; i < XL; ++i) {
    const int row = (wave * XL + i) * 8 + lane / 8, piece = (lane % 8) ^ (row & 7);
    xo[i] = (uint32_t)(m0 + row < g.M ? row : g.M - 1 - m0) * (uint32_t)g.K + piece * 16;
  }
#pragma unroll
  for (int i = 0; i < WL; ++i) {
    const int row = (wave * WL + i) * 16 + lane / 4, piece = (lane % 4) ^ (row >> 4 & 3);
    wo[i] = (uint32_t)(n0 + row < g.N ? row : g.N - 1 - n0) * (uint32_t)(g.K / 2) + piece * 16;
  }
  const int sl = wave % SL;                     // waves beyond the scales' loads bring some of them once more
  const bool s_x = sl < BM / 64;
  {
    const int row = (s_x ? sl : sl - BM / 64) * 64 + lane, last = s_x ? g.M - 1 - m0 : g.N - 1 - n0;
    so = (uint32_t)(row < last ? row : last) * (uint32_t)z.step;
  }
  const unsigned char* sbase = s_x ? z.xs + (size_t)m0 * z.step : z.ws + (size_t)n0 * z.step;

  uint32_t to_lds = 0;                          // the place of the next step asked for
  const unsigned char *xk = x, *wk = w, *sk = sbase;
  // BULK: a whole step; else one that k may end inside of, or none any more
  const auto ask = [&](auto bulk, int step) {
    constexpr bool BULK = decltype(bulk)::value;
    if (!BULK && step >= steps) return;
    // scales first, so that a wait that counts the operands alone waits for no more than them
    if (step % 4 == 0) mx_to_lds16(sk, so, AT_S + (step & 4) / 4 * GROUP + sl * 1024);
    if (BULK || step < full) {
#pragma unroll
      for (int i = 0; i < XL; ++i) mx_to_lds16(xk, xo[i], to_lds + (wave * XL + i) * 1024);
#pragma unroll
      for (int i = 0; i < WL; ++i) mx_to_lds16(wk, wo[i], to_lds + AT_W + (wave * WL + i) * 1024);
    } else {
      // k ends inside this step: nothing behind it, zero in x, any codes in w
#pragma unroll
      for (int i = 0; i < XL; ++i) {
        const int row = (wave * XL + i) * 8 + lane / 8, piece = (lane % 8) ^ (row & 7);
        if (step * 8 + piece < pieces) mx_to_lds16(xk, xo[i], to_lds + (wave * XL + i) * 1024);
        else reinterpret_cast<mx_u32x4*>(mx_lds + to_lds + (wave * XL + i) * 1024)[lane] = mx_u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int i = 0; i < WL; ++i) {
        const int row = (wave * WL + i) * 16 + lane / 4, piece = (lane % 4) ^ (row >> 4 & 3);
        if (step * 4 + piece < pieces / 2) mx_to_lds16(wk, wo[i], to_lds + AT_W + (wave * WL + i) * 1024);
      }
    }
    xk += 128;
    wk += 64;
    sk += 4;
    to_lds = to_lds == (NS - 1) * STAGE ? 0 : to_lds + STAGE;
  };

  mx_f32x4 acc[TM][4];
#pragma unroll
  for (int m = 0; m < TM; ++m)
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[m][t] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
  // With eight tiles of rows a wave, the second four are read while the first are multiplied, each in the registers that it frees
  constexpr int HELD = TM > 4 ? 4 : TM;
  static_assert(HELD == TM || KG == 1, "a step's place stays while it is multiplied");
  mx_i32x8 wf[4], xf[HELD];
  int ws[4], xs[HELD];
  // where a lane reads: the tiles lie a fixed number of bytes apart
  const uint32_t w_at = AT_W + (wn * 64 + 16 * (r / 4) + r % 4) * 64 + (q ^ (r / 4)) * 16;
  const uint32_t x_at = (wm * TM * 16 + r) * 128 + (q ^ (r & 7)) * 16;
  const uint32_t ws_at = AT_S + (BM + wn * 64 + 16 * (r / 4) + r % 4) * 16 + q, xs_at = AT_S + (wm * TM * 16 + r) * 16 + q;
  uint32_t from = KG == 2 && group ? STAGE : 0;  // the place of the step to read
  const unsigned char *wl, *x0, *x1, *wsl, *xsl;
  const auto read_x = [&](int m) {
    const mx_u32x4 lo = *reinterpret_cast<const mx_u32x4*>(x0 + m * 2048), hi = *reinterpret_cast<const mx_u32x4*>(x1 + m * 2048);
    xf[m % HELD] = mx_i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
    xs[m % HELD] = xsl[m * 256];
  };
  const auto read = [&](int step) {
    const uint32_t sc = (step & 4) / 4 * GROUP + (step & 3) * 4;
    wl = mx_lds + (w_at + from);
    x0 = mx_lds + (x_at + from);
    x1 = mx_lds + ((x_at ^ 64) + from);
    wsl = mx_lds + (ws_at + sc);
    xsl = mx_lds + (xs_at + sc);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const mx_u32x4 v = *reinterpret_cast<const mx_u32x4*>(wl + t * 256);
      wf[t] = mx_i32x8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0};
      ws[t] = wsl[t * 64];
    }
#pragma unroll
    for (int m = 0; m < HELD; ++m) read_x(m);
    from += KG * STAGE;
    from = from >= NS * STAGE ? from - NS * STAGE : from;
  };
  const auto multiply = [&]() {
#pragma unroll
    for (int m = 0; m < TM; ++m) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
        acc[m][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[t], xf[m % HELD], acc[m][t], 4, 0, 0, ws[t], 0, xs[m % HELD]);
      if (m + HELD < TM) read_x(m + HELD);
    }
  };
  // the end of a phase; `waits`: for the step that the next one reads, with NS - 2 whole ones asked for behind it, or for all
  const auto end = [&](bool waits, bool all) {
    if (waits) {
      if (all) ta_wait_loads<0>();
      else ta_wait_loads<(NS - 2) * LOADS>();
    }
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  const std::integral_constant<bool, true> inside{};
  const std::integral_constant<bool, false> any{};

#pragma unroll
  for (int i = 0; i < NS - 1; ++i) ask(any, i);
  end(true, NS - 1 >= full);
  if (KG == 1) {
    // phases 2 k and 2 k + 1: group 0 reads step k, then multiplies; group 1 multiplies step k - 1, then reads step k; in the
    // second both ask
    int k = 0;
    if (group) {
      end(false, false);
      for (; k + NS <= full; ++k) {
        ask(inside, k + NS - 1);
        read(k);
        end(true, false);
        multiply();
        end(false, false);
      }
      for (; k < steps; ++k) {
        ask(any, k + NS - 1);
        read(k);
        end(true, true);
        multiply();
        end(false, false);
      }
    } else {
      for (; k + NS <= full; ++k) {
        read(k);
        end(false, false);
        ask(inside, k + NS - 1);
        multiply();
        end(true, false);
      }
      for (; k < steps; ++k) {
        read(k);
        end(false, false);
        ask(any, k + NS - 1);
        multiply();
        end(true, true);
      }
      end(false, false);
    }
  } else {
    // phase p: the group p % 2 reads step p, the other multiplies step p - 1, both ask
    int p = 0;
    if (group) {
      ask(any, NS - 1);
      end(true, NS > full);
      p = 1;
    }
    for (; p + NS + 1 <= full; p += 2) {
      ask(inside, p + NS - 1);
      read(p);
      end(true, false);
      ask(inside, p + NS);
      multiply();
      end(true, false);
    }
    for (; p < steps; p += 2) {
      ask(any, p + NS - 1);
      read(p);
      end(true, true);
      ask(any, p + NS);
      multiply();
      end(true, true);
    }
    if (p == steps) end(true, true);             // as many phases for either group: the last of them was the other's
  }
  ta_wait_loads<0>();

  if (KG == 2) {
    // the second group's sums through LDS: nobody reads steps or loads them any more
    asm volatile("s_barrier" ::: "memory");
    mx_f32x4* sums = reinterpret_cast<mx_f32x4*>(mx_lds);
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if (group) sums[((part * TM + m) * 4 + t) * 64 + lane] = acc[m][t];
      }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (group) return;
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
      for (int t = 0; t < 4; ++t) acc[m][t] += sums[((part * TM + m) * 4 + t) * 64 + lane];
  }

  const int n = n0 + wn * 64 + 16 * q;           // this lane's 16 columns
  float add[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) add[i] = g.bias && n + i < g.N ? g.bias[n + i] : 0.f;
  const bool whole = n + 16 <= g.N && g.ldo % 8 == 0 && (uintptr_t)g.out % 16 == 0;
#pragma unroll
  for (int m = 0; m < TM; ++m) {
    const int row = m0 + (wm * TM + m) * 16 + r;
    if (row >= g.M) continue;
    bf16_t* o = (bf16_t*)g.out + row * g.ldo + n;
    if (whole) {
      mx_u32x4 v[2];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          v[t / 2][t % 2 * 2 + i] =
              f32x2_to_bf16x2_bits(acc[m][t][2 * i] + add[4 * t + 2 * i], acc[m][t][2 * i + 1] + add[4 * t + 2 * i + 1]);
      reinterpret_cast<mx_u32x4*>(o)[0] = v[0];
      reinterpret_cast<mx_u32x4*>(o)[1] = v[1];
    } else {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n + 4 * t + i < g.N) o[4 * t + i] = from_f32<bf16_t>(acc[m][t][i] + add[4 * t + i]);
    }
  }
}

// scales of rows of `blocks` bytes into rows of `step`, 127 behind them: k that is no multiple of 512 leaves rows off the 16
// bytes that a load to LDS brings
__global__ __launch_bounds__(256) void mx_scales_kernel(const uint8_t* __restrict__ x, const uint8_t* __restrict__ w, uint8_t* __restrict__ to,
                                                        long long m, long long rows, int blocks, int step) {
  const long long at = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  const long long row = at / step;
  const int b = (int)(at % step);
  if (row >= rows) return;
  const uint8_t* from = row < m ? x + row * blocks : w + (row - m) * blocks;
  uint32_t v = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) v |= (uint32_t)(b + i < blocks ? from[b + i] : 127) << (8 * i);
  *reinterpret_cast<uint32_t*>(to + at) = v;
}

template <int BM, int BN, int WM, int WN, int KG, int NS>
static int mx_tile_launch(const char* what, hipStream_t stream, const MxGemm& g, MxTiles z) {
  constexpr int steps = NS * (BM * 128 + BN * 64) + 2 * (BM + BN) * 16, sums = KG == 2 ? BM * BN * 4 : 0;
  constexpr int bytes = steps > sums ? steps : sums;
  static_assert(bytes <= MX_LDS, "a workgroup's LDS");
  const auto kernel = mx_tile_kernel<BM, BN, WM, WN, KG, NS>;
  static bool asked = false;
  if (!asked && bytes > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return ta_fail("%s: %d bytes of LDS refused (%s)", what, bytes, hipGetErrorString(e));
    asked = true;
  }
  z.m_tiles = (g.M + BM - 1) / BM;
  z.n_tiles = (g.N + BN - 1) / BN;
  kernel<<<z.m_tiles * z.n_tiles, 512, bytes, stream>>>(g, z);
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

// 8-bit rows, codes [M][K] and bytes [M][K/32]; out bfloat16. scratch: ta_gemm_mx4_mx8_scratch bytes on 16 (0: null will do
// where the scales start on 16 bytes).
#define MX_FEW_ROWS8 64
static int mx_step(int K) { return (K + 511) / 512 * 16; }
extern "C" long long ta_gemm_mx4_mx8_scratch(int M, int N, int K) {
  return M > MX_FEW_ROWS8 && (K % 512 != 0) ? ((long long)M + N) * mx_step(K) : 0;
}
extern "C" int ta_gemm_mx4_mx8(hipStream_t stream, const void* x, const void* xs, const void* codes, const void* scales, const float* bias,
                               void* out, long long ldo, int M, int N, int K, void* scratch, long long scratch_bytes) {
  static const char what[] = "ta_gemm_mx4_mx8";
  const MxGemm g = {x, (const uint8_t*)xs, (const uint8_t*)codes, (const uint8_t*)scales, bias, out, K, ldo, M, N, K, 0};
  if (mx_gemm_check(what, g)) return 1;
  TA_REQUIRE(K <= 1 << 23, "%s: k %d: at most 8,388,608", what, K);         // 256 rows within 31 bits
  if (M == 0) return 0;
  if (M <= 1) return mx_few_launch<true, false, 1, 1, 4, 1>(what, stream, g);
  if (M <= 4) return mx_few_launch<true, false, 1, 1, 4, 4>(what, stream, g);
  if (M <= 8) return mx_few_launch<true, false, 1, 1, 4, 8>(what, stream, g);
  if (M <= 16) return mx_few_launch<true, false, 1, 1, 4, 16>(what, stream, g);
  if (M <= 32) return mx_few_launch<true, false, 2, 2, 2, 32>(what, stream, g);
  if (M <= MX_FEW_ROWS8) return mx_few_launch<true, false, 4, 2, 2, 64>(what, stream, g);
  MxTiles z = {g.xs, g.scales, K / MX_BLOCK, 0, 0};
  if (K % 512 || (uintptr_t)xs % 16 || (uintptr_t)scales % 16) {
    z.step = mx_step(K);
    const long long need = ((long long)M + N) * z.step, grid = (need / 4 + 255) / 256;
    TA_REQUIRE(scratch && scratch_bytes >= need && (uintptr_t)scratch % 16 == 0, "%s: %lld bytes of scratch, %lld are needed", what,
               scratch ? scratch_bytes : 0LL, need);
    TA_REQUIRE(grid <= 0x7fffffffLL, "%s: M=%d N=%d K=%d: more scales than a launch holds", what, M, N, K);
    mx_scales_kernel<<<(int)grid, 256, 0, stream>>>(g.xs, g.scales, (uint8_t*)scratch, M, (long long)M + N, K / MX_BLOCK, z.step);
    if (ta_check_launch(what)) return 1;
    z.xs = (const uint8_t*)scratch;
    z.ws = z.xs + (size_t)M * z.step;
  }
  const long long big = (((long long)M + 255) / 256) * (((long long)N + 255) / 256);
  const long long mid = (((long long)M + 127) / 128) * (((long long)N + 127) / 128);
  if (const char* e = getenv("MXT")) switch (atoi(e)) {
    case 1: return mx_tile_launch<64, 128, 2, 2, 2, 3>(what, stream, g, z);
    case 2: return mx_tile_launch<64, 128, 2, 2, 2, 4>(what, stream, g, z);
    case 4: return mx_tile_launch<128, 128, 2, 2, 2, 3>(what, stream, g, z);
    case 5: return mx_tile_launch<128, 128, 2, 2, 2, 4>(what, stream, g, z);
    case 6: return mx_tile_launch<128, 256, 2, 4, 1, 3>(what, stream, g, z);
    case 8: return mx_tile_launch<256, 256, 2, 4, 1, 3>(what, stream, g, z);
    case 9: return mx_tile_launch<256, 128, 4, 2, 1, 3>(what, stream, g, z);
    case 11: return mx_tile_launch<128, 128, 4, 2, 1, 3>(what, stream, g, z);
    case 12: return mx_tile_launch<64, 128, 4, 2, 1, 4>(what, stream, g, z);
  }
  if (big >= 256) return mx_tile_launch<256, 256, 2, 4, 1, 3>(what, stream, g, z);
  if (mid >= 256) return mx_tile_launch<128, 128, 2, 2, 2, 3>(what, stream, g, z);
  return mx_tile_launch<64, 128, 2, 2, 2, 3>(what, stream, g, z);
}
