// out[m, n] = sum over k of x[m, k] w[n, k] with 4-bit weights (mx.h), x in bfloat16 or in 8-bit blocks.
//
// bfloat16 rows: a power of two times an e2m1 value is a bfloat16, so the codes are widened exactly
// (v_cvt_scalef32_pk_bf16_fp4, two an instruction, scale included) and the products run on v_mfma_f32_16x16x32_bf16 with
// float32 sums.
//
// 8-bit rows: v_mfma_scale_f32_16x16x128_f8f6f4 takes both operands and both scales as they are. It lines up the 128 products
// of a call to the largest one's exponent before it adds them, which leaves some 15 bits below it; from call to call sums are
// float32. Measured on normal weights and normed rows (64 x 4,096 over k = 14,336): the sums are off by 6.8e-6 of the root of their
// products' sum of squares (5e-5 at most, no bias), where float32 sums are off by 4e-8. Beside a result's size that is some 1/240 of
// bfloat16's rounding, 1.65e-3: 0.6 % of the results round to the neighbour, and the results as a whole are as far from 64 bits
// as rounded float32 sums are, 1.6536e-3. So they leave as bfloat16 only; one result in 500, which cancels to little beside its
// products, is off by more than a bfloat16's half step of itself (as it is, by far more, from the rows' rounding to 4 bits).
//
// Times below are GPU time a call inside a graph, weights out of memory; two forms compared were measured in turn.
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

// Results go out in wide stores whatever the row's length leaves of their alignment (1,638 x 2,518 over k = 704, rows on 4 bytes, with operands
// in the caches 12.4 us; 16.3 a row at a time through LDS, 29 single)
typedef mx_f32x4 mx_f32x4_any __attribute__((aligned(4)));
typedef mx_u32x4 mx_u32x4_any __attribute__((aligned(2)));
typedef mx_u32x2 mx_u32x2_any __attribute__((aligned(2)));

// COUNT neighbouring results of a row at out + at, `left` of them inside it; whole: all
template <int COUNT>
__device__ __forceinline__ void mx_store(const MxGemm& g, long long at, const float* y, bool whole, int left) {
  if (g.wide) {
    float* o = (float*)g.out + at;
    if (whole) {
#pragma unroll
      for (int i = 0; i < COUNT; i += 4) *reinterpret_cast<mx_f32x4_any*>(o + i) = mx_f32x4{y[i], y[i + 1], y[i + 2], y[i + 3]};
    } else {
#pragma unroll
      for (int i = 0; i < COUNT; ++i)
        if (i < left) o[i] = y[i];
    }
    return;
  }
  bf16_t* o = (bf16_t*)g.out + at;
  if (whole) {
#pragma unroll
    for (int i = 0; i < COUNT; i += COUNT < 8 ? 4 : 8) {
      if (COUNT < 8) {
        *reinterpret_cast<mx_u32x2_any*>(o + i) = mx_u32x2{f32x2_to_bf16x2_bits(y[i], y[i + 1]), f32x2_to_bf16x2_bits(y[i + 2], y[i + 3])};
      } else {
        mx_u32x4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = f32x2_to_bf16x2_bits(y[(i + 2 * j) % COUNT], y[(i + 2 * j + 1) % COUNT]);
        *reinterpret_cast<mx_u32x4_any*>(o + i) = v;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < COUNT; ++i)
      if (i < left) o[i] = from_f32<bf16_t>(y[i]);
  }
}

// ---------------------------------------------------------------- few rows
// A workgroup owns 16 rows of the weights (or 32, T 2; with GLU 16 gates and their ups) and up to 16 rows of x; its waves deal k out among
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
// busy with; fewer than four a workgroup leave too many of the sums' exchanges. LDS may hold fewer: 8 bfloat16 rows in chunks of 512
// take 16 KB a wave, so ten.
//
// Measured: 8-bit rows, 1 x 28,672 x 4,096 12.6 us (5.0 TB/s of a copy's 5.1), 8 x 14,336 x 4,096 10.7, 16 rows 11.3, where x
// through LDS costs as much as the weights; bfloat16 rows 1 x 4,096 x 4,096 4.6 (launch, one way to memory, the sums), 1 x 4,096 x 14,336
// 8.4, 8 x 4,096 x 14,336 11.8, gated 1 x 14,336 x 4,096 15.4 (4.1 TB/s: an instruction for every two codes).
template <bool X8, bool GLU, int S, int R, int T>
__global__ __launch_bounds__(1024) void mx_few_kernel(MxGemm g, int bytes) {
  if (gridDim.y > 1) {                          // this workgroup's R rows
    const long long at = (long long)blockIdx.y * R;
    g.x = (const unsigned char*)g.x + at * g.ldx * (X8 ? 1 : 2);
    if (X8) g.xs += at * (g.K / MX_BLOCK);
    g.out = (unsigned char*)g.out + at * g.ldo * (g.wide ? 4 : 2);
    g.M = g.M - (int)at < R ? g.M - (int)at : R;
  }
  static_assert(R <= 16 && (S == 2 || S == 4), "rows of a tile, loads in pairs");
  constexpr int P = (X8 ? 8 : 16) * S;          // 16-byte pieces of a row of x in a chunk
  constexpr int FLIP = P < 16 ? P - 1 : 15;
  constexpr int NT = GLU ? 2 : T;               // tiles of the weights: gates and ups, or neighbours
  static_assert(!GLU || T == 1, "16 gates");
  constexpr int XI = R * P > 64 ? R * P / 64 : 1;               // loads of x
  constexpr int LOADS = XI + NT * (S + 1) + (X8 ? 1 : 0);       // of a chunk: at least so many
  extern __shared__ __attribute__((aligned(16))) unsigned char mx_lds[];
  // (what is the same in a whole wave is told to be: addresses are then one base and 32 bits a lane)
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, r = lane % 16, q = lane / 16,
            waves = blockDim.x / 64;
  const int n0 = blockIdx.x * (16 * T), blocks = g.K / MX_BLOCK, chunks = blocks / (4 * S);
  unsigned char* mine = mx_lds + wave * bytes;
  const uint8_t *codes[NT], *scales[NT];        // of the workgroup's first row, of its first ups
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    codes[t] = g.codes + ((size_t)n0 + (GLU && t ? (size_t)g.N : 0)) * (g.K / 2);
    scales[t] = g.scales + ((size_t)n0 + (GLU && t ? (size_t)g.N : 0)) * blocks;
  }
  uint32_t col[T];                              // this lane's rows of the weights, from n0 on
  uint32_t piece_at[T][2];                      // what it loads: a block of row r % 8, of row 8 + r % 8
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const int last = g.N - 1 - n0;
    col[t] = 16 * t + r < last ? 16 * t + r : last;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = 16 * t + 8 * h + r % 8;
      piece_at[t][h] = (uint32_t)(at < last ? at : last) * (uint32_t)(g.K / 2) + (q + 4 * (r / 8)) * 16;
    }
  }
  const uint32_t row = r < g.M ? r : g.M - 1;   // and of x
  const uint32_t xstep = (uint32_t)g.ldx * (X8 ? 1 : 2);
  mx_f32x4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
  mx_u32x4 w[2][NT][S];
  uint32_t ws[2][NT][S], xs[2][S];

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
    if (X8) __builtin_memcpy(xs[set], g.xs + (size_t)c * 4 * S + row * (uint32_t)blocks, 4 * S);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      __builtin_memcpy(ws[set][t], scales[t] + (size_t)c * 4 * S + col[t % T] * (uint32_t)blocks, 4 * S);
#pragma unroll
      for (int s = 0; s < S; ++s)
        w[set][t][s] = __builtin_nontemporal_load(
            reinterpret_cast<const mx_u32x4*>(codes[t] + (size_t)(c * S + s / 2 * 2) * 64 + piece_at[t % T][s % 2]));
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
    const auto piece = [&](int p) {
      return *reinterpret_cast<const mx_u32x4*>(xl + (row * P + (p ^ (row & FLIP))) * 16);
    };
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (X8) {
        // lane group q holds the halves q % 2 of the 128 k's blocks q / 2 and 2 + q / 2, and block q's scale
        const mx_u32x4 lo = piece(8 * s + q), hi = piece(8 * s + 4 + q);
        const mx_i32x8 a = {(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const mx_u32x4 c = w[set][t][s];
          const mx_i32x8 b = {(int)c[0], (int)c[1], (int)c[2], (int)c[3], 0, 0, 0, 0};
          acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc[t], 0, 4, 0, (int)(xs[set][s] >> (8 * q)), 0,
                                                                    (int)(ws[set][t][s] >> (8 * q)));
        }
      } else {
        mx_bf16x8 a[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = __builtin_bit_cast(mx_bf16x8, piece(16 * s + 4 * q + j));
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float scale = mx_scale(ws[set][t][s] >> (8 * q) & 255u);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[j], mx_widen8(w[set][t][s][j], scale), acc[t], 0, 0, 0);
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
          w[0][t][s] = *reinterpret_cast<const mx_u32x4*>(codes[t] + (size_t)b * 16 + col[t % T] * (uint32_t)(g.K / 2));
          ws[0][t][s] = (uint32_t)scales[t][b + col[t % T] * (uint32_t)blocks] * 0x01010101u;
        }
      }
      if (X8) xs[0][s] = live ? (uint32_t)g.xs[b + row * (uint32_t)blocks] * 0x01010101u : 0x7f7f7f7fu;
    }
    multiply(0);
  }
  // the sums, in the place of the wave's x
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  float* part = reinterpret_cast<float*>(mine);
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[t * 256 + (q * 4 + i) * 16 + r] = acc[t][i];
  __syncthreads();
  for (int at = threadIdx.x; at < 256 * T; at += blockDim.x) {
    const int m = at % 256 / 16, n = n0 + at / 256 * 16 + at % 16;
    if (m >= g.M || n >= g.N) continue;
    float v[GLU ? 2 : 1];
#pragma unroll
    for (int t = 0; t < (GLU ? 2 : 1); ++t) {
      v[t] = 0.f;
      for (int wv = 0; wv < waves; ++wv) v[t] += reinterpret_cast<const float*>(mx_lds + wv * bytes)[t * 256 + at];
      if (g.bias) v[t] += g.bias[n + (long long)t * g.N];
    }
    const float y = GLU ? v[0] / (1.0f + expf(-v[0])) * v[GLU ? 1 : 0] : v[0];
    const long long to = (long long)m * g.ldo + n;
    if (g.wide) reinterpret_cast<float*>(g.out)[to] = y;
    else reinterpret_cast<bf16_t*>(g.out)[to] = from_f32<bf16_t>(y);
  }
}

#define MX_LDS (160 * 1024)
// A launch counts its threads in 32 bits and loses what is beyond without an error. Rows that would be too many go out in several launches
// (MX_ROWS), columns are refused.
#define MX_ROWS (1 << 26)
static bool mx_launch_holds(long long groups, int threads) { return groups * threads <= 0xffffffffLL; }

template <bool X8, bool GLU, int S, int R, int T = 1>
static int mx_few_launch(const char* what, hipStream_t stream, const MxGemm& g) {
  constexpr int x = R * (X8 ? 8 : 16) * S * 16, sums = (GLU ? 2 : T) * 1024;
  const auto kernel = mx_few_kernel<X8, GLU, S, R, T>;
  const int chunks = g.K / (128 * S), grid = (int)(((long long)g.N + 16 * T - 1) / (16 * T));
  // as many waves as give every CU 16, then the fewest that need as many turns; one buffer of x does for one turn
  int waves = (16 * 256 + grid - 1) / grid;
  waves = waves < 4 ? 4 : waves > 16 ? 16 : waves;
  if (waves > chunks) waves = chunks > 0 ? chunks : 1;
  int bytes = waves < chunks ? 2 * x : x;
  if (bytes < sums) bytes = sums;
  if (waves * bytes > MX_LDS) {
    bytes = 2 * x > sums ? 2 * x : sums;
    waves = MX_LDS / bytes;
  }
  const int turns = (chunks + waves - 1) / waves;
  if (turns > 0) waves = (chunks + turns - 1) / turns;
  TA_REQUIRE(mx_launch_holds(grid, waves * 64), "%s: M=%d N=%d are more than a launch holds", what, g.M, g.N);
  static int allowed = 64 * 1024;
  if (waves * bytes > allowed) {
    const hipError_t e =
        hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, MX_LDS);
    if (e != hipSuccess) return ta_fail("%s: %d bytes of LDS refused (%s)", what, MX_LDS, hipGetErrorString(e));
    allowed = MX_LDS;
  }
  kernel<<<dim3(grid, (g.M + R - 1) / R), waves * 64, (size_t)waves * bytes, stream>>>(g, bytes);
  return ta_check_launch(what);
}

// ---------------------------------------------------------------- tiles of many rows
// Tiles of BM rows by BN rows of the weights, k by steps of 128 (one scaled matrix instruction, or four on bfloat16). Both operands
// come into LDS without registers in between, NS - 1 steps ahead, and so do the scales of every four steps (a row's are four bytes a
// step in a line of their own: step by step they cost as many requests as the operands).
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
// Pieces of 16 bytes are permuted by the row's number, so that the addresses of sixteen lanes (one q) meet every bank once. The counters
// still have 1.25 cycles of bank conflicts for each LDS instruction of the 256 x 256 tile, of 4.5 that it takes; what they come from is
// not known.
// Measured: a step of 64 x 128 takes 0.33 us with operands in the caches (0.45 out of memory), of 256 x 256 1.6, where the matrix
// instructions alone need 0.13 and 1.0, the way into LDS 0.11 and 0.33 and the reads 0.11 and 0.5: the small tile's parts add up and do not
// overlap. 4,096 x 28,672 x 4,096 375 us (2.6 PFLOP/s of the instruction's 4.2), 512 x 4,096 x 14,336 50 (38 to 42 in the caches).
// Where the tiles do not fill the CUs, k is cut among `parts` workgroups, which leave float32 sums in planes; mx_planes_kernel adds
// them in order and finishes. GLU: a tile holds 64 gates and their 64 ups, a lane's 16 columns are then 8 of either.
__device__ __host__ __forceinline__ long long mx_pad(int n) { return (n + 3LL) / 4 * 4; }
struct MxTiles {
  const uint8_t *xs, *ws;     // scales in rows of `step` bytes, a multiple of 16, 127 behind the last block; step 0: as they are, rows
  int step;                   // that do not start on 16 bytes, all of a part's brought through registers in front of its steps
  int m_tiles, n_tiles;
  int parts, part_steps;      // steps of a part, a multiple of 4
  float* planes;              // [parts][M][mx_pad(N), with GLU twice], or null
};

// 16 bytes a lane to the LDS that starts at `lds`; base and lds are the whole wave's
__device__ __forceinline__ void mx_to_lds16(const void* base, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(lds) : "m0", "memory");
}

// which of a row's pieces lie where: sixteen rows' addresses of a piece have every bank once, two rows of 8 pieces (of 256 bytes
// together) or one of 16 in each of the places that a bank has
template <bool X8>
__device__ __forceinline__ uint32_t mx_flip(uint32_t row) {
  return X8 ? row >> 1 & 7 : row & 15;
}

template <bool X8, bool GLU, int BM, int BN, int WM, int WN, int KG, int NS>
__global__ __launch_bounds__(512) void mx_tile_kernel(MxGemm g, MxTiles z) {
  constexpr int W = 8, TM = BM / (16 * WM), XB = X8 ? 128 : 256;        // bytes of a row of x in a step
  constexpr int XP = XB / 16;                                           // its pieces
  constexpr int XL = BM * XB / 1024 / W, WL = BN / 16 / W;     // loads of 1 KB a wave and step
  constexpr int SX = X8 ? BM : 0, SL = (SX + BN) / 64;         // loads of 64 rows' scales, one a wave
  constexpr int LOADS = XL + WL;
  constexpr int AT_W = BM * XB, STAGE = AT_W + BN * 64, AT_S = NS * STAGE, GROUP = (SX + BN) * 16;
  static_assert(BN == 64 * WN && WM * WN * KG == W && BM % (16 * WM) == 0, "eight waves");
  static_assert(XL * 1024 * W == BM * XB && WL * 16 * W == BN && SL <= W && NS <= 4, "tiles in whole loads");
  extern __shared__ __attribute__((aligned(16))) unsigned char mx_lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, r = lane % 16, q = lane / 16;
  const int group = wave / 4, part = KG == 2 ? wave % 4 : wave, wm = part / WN, wn = part % WN;
  // workgroups go round the 8 XCDs: each gets neighbouring tiles, all rows of a band of columns, so that its cache holds them
  const int tiles = z.m_tiles * z.n_tiles, per = tiles / 8, b = blockIdx.x % tiles, cut = blockIdx.x / tiles;
  const int tile = b < per * 8 ? (b % 8) * per + b / 8 : b;
  // bands of four tiles of rows, columns after columns inside a band: the 32 tiles that an XCD has under way then read a quarter of
  // the rows and eight columns' weights and not all rows
  const int band = tile / (4 * z.n_tiles), in = tile % (4 * z.n_tiles), high = z.m_tiles - 4 * band < 4 ? z.m_tiles - 4 * band : 4;
  const int m0 = (4 * band + in % high) * BM, n0 = in / high * (GLU ? BN / 2 : BN);
  const int first = cut * z.part_steps, left = (g.K + 127) / 128 - first;       // this part's steps
  const int steps = left < z.part_steps ? left : z.part_steps;
  const int whole_steps = g.K / 128 - first, full = whole_steps < steps ? whole_steps : steps;
  const int pieces = g.K / (X8 ? 16 : 8) - first * XP, wpieces = g.K / 32 - first * 4;
  const unsigned char* x = (const unsigned char*)g.x + (size_t)m0 * g.ldx * (X8 ? 1 : 2) + (size_t)first * XB;
  const unsigned char* w = g.codes + (size_t)n0 * (g.K / 2) + (size_t)first * 64;

  uint32_t xo[XL], wo[WL], so;
#pragma unroll
  for (int i = 0; i < XL; ++i) {
    const int at = (wave * XL + i) * 64 + lane, row = at / XP, piece = (at % XP) ^ mx_flip<X8>(row);
    xo[i] = (uint32_t)(m0 + row < g.M ? row : g.M - 1 - m0) * ((uint32_t)g.ldx * (X8 ? 1 : 2)) + piece * 16;
  }
  // row of the weights, from n0 on, behind row `row` of the tile
  const auto weight_row = [&](int row) {
    if (!GLU) return (uint32_t)(n0 + row < g.N ? row : g.N - 1 - n0);
    const int c = row / 64 * 32 + row % 64 / 16 * 8 + row % 8, up = row % 16 / 8;
    return (uint32_t)(n0 + c < g.N ? c : g.N - 1 - n0) + (up ? (uint32_t)g.N : 0u);
  };
#pragma unroll
  for (int i = 0; i < WL; ++i) {
    const int row = (wave * WL + i) * 16 + lane / 4, piece = (lane % 4) ^ (row >> 4 & 3);
    wo[i] = weight_row(row) * (uint32_t)(g.K / 2) + piece * 16;
  }
  const int sl = wave % SL;                     // waves beyond the scales' loads bring some of them once more
  const bool s_x = sl < SX / 64;
  {
    // (16-byte places: of every 64 rows' scales, those that a wave reads at once, 16 apart, lie in different banks)
    const int row = (s_x ? sl : sl - SX / 64) * 64 + (lane ^ (lane >> 4 & 3) * 4);
    so = (s_x ? (uint32_t)(m0 + row < g.M ? row : g.M - 1 - m0) : weight_row(row)) * (uint32_t)z.step;
  }
  const unsigned char* sbase = (s_x ? z.xs + (size_t)m0 * z.step : z.ws + (size_t)n0 * z.step) + (size_t)first * 4;

  uint32_t to_lds = 0;                          // the place of the next step asked for
  const unsigned char *xk = x, *wk = w, *sk = sbase;
  // a whole step's loads, one by one: scales first, so that a wait that counts the operands alone waits for no more than them
  const auto ask_one = [&](int step, int i) {
    if (i == 0 && step % 4 == 0 && z.step) mx_to_lds16(sk, so, AT_S + (step & 4) / 4 * GROUP + sl * 1024);
    if (i < XL) mx_to_lds16(xk, xo[i < XL ? i : 0], to_lds + (wave * XL + i) * 1024);
    else mx_to_lds16(wk, wo[i >= XL ? i - XL : 0], to_lds + AT_W + (wave * WL + i - XL) * 1024);
  };
  const auto asked = [&]() {
    xk += XB;
    wk += 64;
    sk += 4;
    to_lds = to_lds == (NS - 1) * STAGE ? 0 : to_lds + STAGE;
  };
  const auto ask_all = [&](int step) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) ask_one(step, i);
    asked();
  };
  // a step that k may end inside of, or none any more
  const auto ask = [&](int step) {
    if (step >= steps) return;
    if (step < full) {
      ask_all(step);
      return;
    } else {
      // k ends inside this step: nothing behind it, zero in x, any codes in w
      if (step % 4 == 0 && z.step) mx_to_lds16(sk, so, AT_S + (step & 4) / 4 * GROUP + sl * 1024);
#pragma unroll
      for (int i = 0; i < XL; ++i) {
        const int at = (wave * XL + i) * 64 + lane, row = at / XP, piece = (at % XP) ^ mx_flip<X8>(row);
        if (step * XP + piece < pieces) mx_to_lds16(xk, xo[i], to_lds + (wave * XL + i) * 1024);
        else reinterpret_cast<mx_u32x4*>(mx_lds + to_lds + (wave * XL + i) * 1024)[lane] = mx_u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int i = 0; i < WL; ++i) {
        const int row = (wave * WL + i) * 16 + lane / 4, piece = (lane % 4) ^ (row >> 4 & 3);
        if (step * 4 + piece < wpieces) mx_to_lds16(wk, wo[i], to_lds + AT_W + (wave * WL + i) * 1024);
      }
    }
    asked();
  };

  mx_f32x4 acc[TM][4];
#pragma unroll
  for (int m = 0; m < TM; ++m)
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[m][t] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
  // With eight tiles of rows a wave, the second four are read while the first are multiplied, each in the registers that it frees
  constexpr int HELD = TM > 4 ? 4 : TM;
  static_assert(HELD == TM || KG == 1, "a step's place stays while it is multiplied");
  mx_u32x4 wf[4], xf[HELD][XP / 4];
  int ws[4], xs[HELD];
  // where a lane reads: the tiles lie a fixed number of bytes apart
  const uint32_t w_at = AT_W + (wn * 64 + 16 * (r / 4) + r % 4) * 64 + (q ^ (r / 4)) * 16;
  const uint32_t x_at = (wm * TM * 16 + r) * XB;
  const uint32_t ws_at = AT_S + (SX + wn * 64 + 16 * (r / 4) + r % 4) * 16 + q, xs_at = AT_S + wm * TM * 256 + q;
  uint32_t from = KG == 2 && group ? STAGE : 0;  // the place of the step to read
  const unsigned char *xl, *xsl;
  const auto read_x = [&](int m) {
#pragma unroll
    for (int i = 0; i < XP / 4; ++i) {
      // 8 bits: halves q % 2 of the blocks q / 2 and 2 + q / 2; bfloat16: the four eights of block q
      const uint32_t piece = X8 ? (uint32_t)(q + 4 * i) ^ mx_flip<X8>(r) : (uint32_t)(4 * q + i) ^ mx_flip<X8>(r);
      xf[m % HELD][i] = *reinterpret_cast<const mx_u32x4*>(xl + piece * 16 + m * 16 * XB);
    }
    if (X8) xs[m % HELD] = xsl[m * 256 + (r ^ ((wm * TM + m) & 3) * 4) * 16];
  };
  const auto read = [&](int step) {
    const uint32_t sc = (z.step ? step >> 2 & 1 : step >> 2) * GROUP + (step & 3) * 4;
    const unsigned char *wl = mx_lds + (w_at + from), *wsl = mx_lds + (ws_at + sc);
    xl = mx_lds + (x_at + from);
    xsl = mx_lds + (xs_at + sc);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      wf[t] = *reinterpret_cast<const mx_u32x4*>(wl + t * 256);
      ws[t] = wsl[(t ^ r / 4) * 64];
    }
#pragma unroll
    for (int m = 0; m < HELD; ++m) read_x(m);
    from += KG * STAGE;
    from = from >= NS * STAGE ? from - NS * STAGE : from;
  };
  // `step`: a whole step whose loads go out between the products (-1: none), where a phase has many: in front of them they keep a wave for
  // as long as the cache takes to accept them (512 x 28,672 x 4,096 58 us so, 55 between; in the small tiles of KG 2 they go out first,
  // 26 and 29 us of 64 rows of bfloat16 against 2 x 14,336 x 4,096: there the way to memory is what a phase waits for)
  const auto multiply = [&](int step) {
    const auto between = [&](int i, int count) {
      if (step >= 0) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j)
          if (j * count / LOADS == i) ask_one(step, j);
      }
      if (KG == 1) __builtin_amdgcn_sched_barrier(0);
    };
    if constexpr (X8) {
#pragma unroll
      for (int m = 0; m < TM; ++m) {
        const mx_u32x4 lo = xf[m % HELD][0], hi = xf[m % HELD][1];
        const mx_i32x8 v = {(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const mx_i32x8 a = {(int)wf[t][0], (int)wf[t][1], (int)wf[t][2], (int)wf[t][3], 0, 0, 0, 0};
          acc[m][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, v, acc[m][t], 4, 0, 0, ws[t], 0, xs[m % HELD]);
        }
        if (KG == 1) __builtin_amdgcn_sched_barrier(0);
        if (m + HELD < TM) read_x(m + HELD);     // here: the compiler would put it right in front of its use
        between(m, TM);
      }
    } else {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float scale = mx_scale((uint32_t)ws[t]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const mx_bf16x8 a = mx_widen8(wf[t][j], scale);
#pragma unroll
          for (int m = 0; m < TM; ++m)
            acc[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(mx_bf16x8, xf[m][j % (XP / 4)]), acc[m][t], 0, 0, 0);
        }
      }
    }
    if (step >= 0) asked();
  };
  // the end of a phase; `next`: the step that has to be there then (none: -1), with whole steps up to `asked` asked for behind it
  const auto end = [&](int next, int asked) {
    if (next >= 0) {
      const int last = asked < full ? asked : full - 1;        // (one that k ends inside of has fewer loads: it does not count)
      if (NS > 3 && last - next >= 2) ta_wait_loads<2 * LOADS>();
      else if (last - next >= 1) ta_wait_loads<LOADS>();
      else ta_wait_loads<0>();
    }
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  const auto end_inside = [&](bool waits) {      // the same with NS - 2 whole steps behind the next
    if (waits) ta_wait_loads<(NS - 2) * LOADS>();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) ask(i);
  if (!z.step) {
    const int blocks = g.K / MX_BLOCK, count = (steps + 3) / 4 * (SX + BN);
    for (int at = threadIdx.x; at < count; at += 4 * 512) {
      mx_u32x4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int place = (at + 512 * j) % (SX + BN), row = place < SX ? place : place - SX, b = (first + (at + 512 * j) / (SX + BN) * 4) * 4;
        const uint8_t* from = place < SX ? z.xs + (size_t)(m0 + row < g.M ? m0 + row : g.M - 1) * blocks
                                         : z.ws + ((size_t)n0 + weight_row(row)) * blocks;
        v[j] = mx_u32x4{0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu};
        if (at + 512 * j >= count) continue;
        if (b + 16 <= blocks) {
          __builtin_memcpy(&v[j], from + b, 16);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (b + i < blocks) v[j][i / 4] = (v[j][i / 4] & ~(255u << (8 * (i % 4)))) | (uint32_t)from[b + i] << (8 * (i % 4));
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int place = (at + 512 * j) % (SX + BN);
        if (at + 512 * j < count)
          *reinterpret_cast<mx_u32x4*>(mx_lds + AT_S + (at + 512 * j) / (SX + BN) * GROUP + (place ^ (place >> 4 & 3) * 4) * 16) = v[j];
      }
    }
  }
  end(0, NS - 2);
  if (KG == 1) {
    // phases 2 k and 2 k + 1: group 0 reads step k, then multiplies; group 1 multiplies step k - 1, then reads step k; in the
    // second both ask
    int k = 0;
    if (group) {
      end(-1, 0);
      for (; k + NS <= full; ++k) {
        read(k);
        ask_all(k + NS - 1);
        end_inside(true);
        multiply(-1);
        end_inside(false);
      }
      for (; k < steps; ++k) {
        read(k);
        ask(k + NS - 1);
        end(k + 1, k + NS - 1);
        multiply(-1);
        end(-1, 0);
      }
    } else {
      for (; k + NS <= full; ++k) {
        read(k);
        end_inside(false);
        multiply(k + NS - 1);
        end_inside(true);
      }
      for (; k < steps; ++k) {
        read(k);
        end(-1, 0);
        ask(k + NS - 1);
        multiply(-1);
        end(k + 1, k + NS - 1);
      }
      end(-1, 0);
    }
  } else {
    // phase p: the group p % 2 reads step p, the other multiplies step p - 1, both ask
    int p = 0;
    if (group) {
      ask(NS - 1);
      end(1, NS - 1);
      p = 1;
    }
    for (; p + NS + 1 <= full; p += 2) {
      ask_all(p + NS - 1);
      read(p);
      end_inside(true);
      ask_all(p + NS);
      multiply(-1);
      end_inside(true);
    }
    for (; p < steps; p += 2) {
      read(p);
      ask(p + NS - 1);
      end(p + 1, p + NS - 1);
      ask(p + NS);
      multiply(-1);
      end(p + 2, p + NS);
    }
    if (p == steps) end(-1, 0);                  // as many phases for either group: the last of them was the other's
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

  if (z.planes) {
    // rows of the weights in this lane's registers: 4 t + i behind the first, with GLU 8 gates and 8 ups
    const long long rows = (GLU ? 2 : 1) * mx_pad(g.N);
    const int n = n0 + (GLU ? wn * 32 + 8 * q : wn * 64 + 16 * q);
#pragma unroll
    for (int m = 0; m < TM; ++m) {
      const int row = m0 + (wm * TM + m) * 16 + r;
      if (row >= g.M) continue;
      float* o = z.planes + ((size_t)cut * g.M + row) * rows + n;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int c = GLU ? 4 * (t % 2) : 4 * t;
        if (n + c < g.N) *reinterpret_cast<mx_f32x4*>(o + c + (GLU && t >= 2 ? mx_pad(g.N) : 0)) = acc[m][t];
      }
    }
    return;
  }
  constexpr int CN = GLU ? 8 : 16;               // this lane's columns of the result
  const int n = n0 + wn * (4 * CN) + CN * q;
  float add[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int c = i % CN;
    add[i] = g.bias && n + c < g.N ? g.bias[n + c + (i >= CN ? (long long)g.N : 0)] : 0.f;
  }
#pragma unroll
  for (int m = 0; m < TM; ++m) {
    const int row = m0 + (wm * TM + m) * 16 + r;
    float y[CN];
#pragma unroll
    for (int i = 0; i < CN; ++i) {
      const float v = acc[m][i / 4][i % 4] + add[i];
      if (GLU) {
        const float u = acc[m][2 + i / 4 % 2][i % 4] + add[8 + i % 8];
        y[i] = v / (1.0f + expf(-v)) * u;
      } else {
        y[i] = v;
      }
    }
    if (row < g.M) mx_store<CN>(g, (long long)row * g.ldo + n, y, n + CN <= g.N, g.N - n);
  }
}

// the planes' sums in order, finished: four columns a thread
template <bool GLU>
__global__ __launch_bounds__(256) void mx_planes_kernel(MxGemm g, const float* __restrict__ planes, int parts) {
  const int per = (g.N + 3) / 4;
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  const int row = (int)(at / per), n = (int)(at % per) * 4;
  if (row >= g.M) return;
  const long long pad = mx_pad(g.N), rows = (GLU ? 2 : 1) * pad, plane = g.M * rows;
  float v[2][4];
#pragma unroll
  for (int u = 0; u < (GLU ? 2 : 1); ++u) {
    const float* p = planes + row * rows + n + u * pad;
    mx_f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int c = 0; c < parts; ++c, p += plane) sum += *reinterpret_cast<const mx_f32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[u][i] = sum[i] + (g.bias && n + i < g.N ? g.bias[n + i + (u ? (long long)g.N : 0)] : 0.f);
  }
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = GLU ? v[0][i] / (1.0f + expf(-v[0][i])) * v[1][i] : v[0][i];
  mx_store<4>(g, (long long)row * g.ldo + n, y, n + 4 <= g.N, g.N - n);
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

template <bool X8, bool GLU, int BM, int BN, int WM, int WN, int KG, int NS>
static int mx_tile_launch(const char* what, hipStream_t stream, const MxGemm& g, MxTiles z) {
  constexpr int steps = NS * (BM * (X8 ? 128 : 256) + BN * 64), scales = ((X8 ? BM : 0) + BN) * 16, sums = KG == 2 ? BM * BN * 4 : 0;
  constexpr int most = steps + (MX_LDS - steps) / scales * scales;
  static_assert(steps >= sums && steps + 2 * scales <= MX_LDS, "a workgroup's LDS");
  const int all = (g.K + 127) / 128, each = z.part_steps < all ? z.part_steps : all;
  const int bytes = steps + (z.step || each <= 8 ? 2 : (each + 3) / 4) * scales;
  TA_REQUIRE(bytes <= most, "%s: scales of %d steps do not fit", what, each);
  const auto kernel = mx_tile_kernel<X8, GLU, BM, BN, WM, WN, KG, NS>;
  static bool asked = false;
  if (!asked) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e != hipSuccess) return ta_fail("%s: %d bytes of LDS refused (%s)", what, most, hipGetErrorString(e));
    asked = true;
  }
  z.m_tiles = (int)(((long long)g.M + BM - 1) / BM);
  z.n_tiles = (int)(((long long)g.N + (GLU ? BN / 2 : BN) - 1) / (GLU ? BN / 2 : BN));
  kernel<<<z.m_tiles * z.n_tiles * z.parts, 512, bytes, stream>>>(g, z);
  return ta_check_launch(what);
}

// What the tiles need: which of them, in how many parts of k, and the bytes of scratch for scales and planes.
struct MxPlan {
  int form;                   // into mx_forms
  int parts, part_steps;
  bool scales;                // laid out again
  long long scale_bytes, bytes;
  double us;
};
// Tiles and what 128 k of one take while every CU has one (measured on MI355X in us: k 4,096 and 14,336, one to seven
// rounds, with the start and the end of a tile spread over its steps). Of 17 shapes the choice is the fastest of all forms and cuts, or within
// 2 %, for 16; 128 x 6,144 over k = 4,096 takes 16.4 us in two parts and 14.0 in one.
static const struct {
  int bm, bn;
  double us;
  int held;                   // steps whose scales LDS holds at once
} mx_forms[] = {{64, 128, 0.40, 64}, {128, 128, 0.62, 64}, {128, 256, 0.93, 40}, {256, 256, 1.60, 8}};
static int mx_step(int K) { return (K + 511) / 512 * 16; }

static MxPlan mx_plan(bool x8, bool glu, int M, int N, int K, bool aligned) {
  const long long rows = glu ? 2LL * N : N;
  const int steps = (K + 127) / 128;
  // scales whose rows do not start on 16 bytes: all of a part's through registers at its start where LDS holds them, else laid out
  // again by a kernel in front, a launch of 2.5 us (323 x 3,347 over k = 4,320: 18.3 and 20.6 us)
  const bool odd = K % 512 != 0 || !aligned;
  MxPlan best = {};
  best.us = 1e30;
  for (int f = 0; f < (x8 ? 4 : 1); ++f) {
    const long long tiles = ((long long)M + mx_forms[f].bm - 1) / mx_forms[f].bm * ((rows + mx_forms[f].bn - 1) / mx_forms[f].bn);
    for (int parts = 1; parts <= 16; ++parts) {
      const int each = ((steps + parts - 1) / parts + 3) / 4 * 4;
      if (parts > 1 && (tiles * parts > 512 || (long long)(parts - 1) * each >= steps)) break;
      // planes are written and read once at some 4 TB/s, by a kernel of their own
      const double planes = parts > 1 ? 2.5 + (double)parts * M * rows * 8 * 0.25e-6 : 0.;
      const bool scales = odd && (each < steps ? each : steps) > mx_forms[f].held;
      const double us = (double)((tiles * parts + 255) / 256) * (each < steps ? each : steps) * mx_forms[f].us * (x8 ? 1. : 1.3) + planes +
                        (scales ? 2.5 : 0.);
      if (us < best.us) best = {f, parts, each, scales, 0, parts > 1 ? parts * (long long)M * (glu ? 2 : 1) * mx_pad(N) * 4 : 0, us};
    }
  }
  best.scale_bytes = best.scales ? ((x8 ? (long long)M : 0) + rows) * mx_step(K) : 0;
  best.bytes += best.scale_bytes;
  return best;
}

template <bool X8, bool GLU>
static int mx_tiles(const char* what, hipStream_t stream, const MxGemm& g, void* scratch, long long scratch_bytes) {
  const bool aligned = (!X8 || (uintptr_t)g.xs % 16 == 0) && (uintptr_t)g.scales % 16 == 0;
  const MxPlan plan = mx_plan(X8, GLU, g.M, g.N, g.K, aligned);
  const long long rows = GLU ? 2LL * g.N : g.N;
  TA_REQUIRE(plan.bytes == 0 || (scratch && scratch_bytes >= plan.bytes && (uintptr_t)scratch % 16 == 0),
             "%s: %lld bytes of scratch, %lld are needed", what, scratch ? scratch_bytes : 0LL, plan.bytes);
  TA_REQUIRE((rows + 256) * (g.K / 2) <= 0xffffffffLL || !GLU, "%s: gates and ups of %d x %d lie more than 4 GB apart", what, g.N, g.K);
  // all launches of the call, before the first
  const auto& form = mx_forms[plan.form];
  const long long xrows = X8 ? g.M : 0, tiles = ((long long)g.M + form.bm - 1) / form.bm * ((rows + form.bn - 1) / form.bn),
                  scales_grid = plan.scales ? ((xrows + rows) * mx_step(g.K) / 4 + 255) / 256 : 0,
                  planes_grid = plan.parts > 1 ? ((long long)g.M * (((long long)g.N + 3) / 4) + 255) / 256 : 0;
  TA_REQUIRE(mx_launch_holds(tiles * plan.parts, 512) && mx_launch_holds(scales_grid, 256) && mx_launch_holds(planes_grid, 256),
             "%s: M=%d N=%d are more than a launch holds", what, g.M, g.N);
  MxTiles z = {g.xs, g.scales, g.K % 512 == 0 && aligned ? g.K / MX_BLOCK : 0, 0, 0, plan.parts, plan.part_steps, nullptr};
  if (plan.scales) {
    z.step = mx_step(g.K);
    mx_scales_kernel<<<(int)scales_grid, 256, 0, stream>>>(g.xs, g.scales, (uint8_t*)scratch, xrows, xrows + rows, g.K / MX_BLOCK, z.step);
    if (ta_check_launch(what)) return 1;
    z.xs = (const uint8_t*)scratch;
    z.ws = z.xs + (size_t)xrows * z.step;
  }
  if (plan.parts > 1) z.planes = (float*)((uint8_t*)scratch + plan.scale_bytes);
  int rc;
  if constexpr (!X8) rc = mx_tile_launch<false, GLU, 64, 128, 2, 2, 2, 4>(what, stream, g, z);
  else if (plan.form == 0) rc = mx_tile_launch<true, false, 64, 128, 2, 2, 2, 4>(what, stream, g, z);
  else if (plan.form == 1) rc = mx_tile_launch<true, false, 128, 128, 2, 2, 2, 3>(what, stream, g, z);
  else if (plan.form == 2) rc = mx_tile_launch<true, false, 128, 256, 2, 4, 1, 3>(what, stream, g, z);
  else rc = mx_tile_launch<true, false, 256, 256, 2, 4, 1, 3>(what, stream, g, z);
  if (rc || plan.parts == 1) return rc;
  mx_planes_kernel<GLU><<<(int)planes_grid, 256, 0, stream>>>(g, z.planes, plan.parts);
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

// What the waves along k take (GPU time in us, measured from 1,024 x 1,024 to 28,672 x 4,096 with 5 to 64 rows): 2.3 and, for every round of
// 256 workgroups and 1,000 k, 0.55 with up to 8 rows of x, 0.68 with up to 16 in 8 bits and 0.88 in bfloat16; with 32 rows of the weights
// (or 16 gates and their ups) a workgroup 0.95, 1.1 and 1.3.
static double mx_few_us(bool x8, bool glu, bool pairs, int M, int N, int K) {
  const int rows = pairs ? 32 : 16;
  const double each = glu || pairs ? (M <= 8 ? 0.95 : x8 ? 1.1 : 1.3) : M <= 8 ? 0.55 : x8 ? 0.68 : 0.88;
  return 2.3 + (double)((((long long)N + rows - 1) / rows * ((M + 15) / 16) + 255) / 256) * each * K * 1e-3;
}

// Whether a workgroup takes 32 rows of the weights and not 16: x then goes through LDS half as often, and there are half as many
// workgroups (64 bfloat16 rows of 4,096 over k = 4,096 12.3 us and 16.0, 16 of 6,144 7.5 and 9.8, 16 of 28,672 22.2 and 26.4; 16 of 4,096,
// where 256 workgroups are one round, 7.4 and 5.7)
static bool mx_few_pairs(bool x8, int M, int N, int K) {
  return M > 4 && mx_few_us(x8, false, true, M, N, K) < 0.97 * mx_few_us(x8, false, false, M, N, K);
}

// Whether the waves along k take it: up to 16 rows always (a step of the 8B shape at batch 8 with 8-bit rows 3,560 tokens a second, with tiles
// for 28,672 columns 3,380: out of memory they come slower); more, in groups of 16 each of which reads the weights again, where that is
// less than what the tiles cost, their steps, planes and scales and 4.5 (32 bfloat16 rows of 4,096 over k = 4,096 7.4 us against 12.7, of
// 14,336 over 4,096 25 against 17).
static bool mx_few(bool x8, bool glu, int M, int N, int K, bool aligned) {
  if (M <= 16) return true;
  if (M > 64) return false;
  double us = mx_few_us(x8, glu, false, M, N, K);
  if (!glu && mx_few_pairs(x8, M, N, K)) us = mx_few_us(x8, false, true, M, N, K);
  return us < mx_plan(x8, glu, M, N, K, aligned).us + 4.5;
}

// Bytes of scratch for M rows in 8 bits (x8) or bfloat16; aligned: all scales start on 16 bytes.
extern "C" long long ta_gemm_mx4_scratch(int x8, int swiglu, int M, int N, int K, int aligned) {
  if (M > MX_ROWS) {
    const long long first = ta_gemm_mx4_scratch(x8, swiglu, MX_ROWS, N, K, aligned), last = ta_gemm_mx4_scratch(x8, swiglu, M % MX_ROWS, N, K, aligned);
    return first > last ? first : last;
  }
  if (M <= 0 || N <= 0 || K < MX_BLOCK || mx_few(x8, swiglu, M, N, K, aligned)) return 0;
  return mx_plan(x8, swiglu, M, N, K, aligned).bytes;
}

// bfloat16 rows x [M][ldx] (rows on 16 bytes), at most ta_mx4_max_rows of them; out_dtype float32 or bfloat16; swiglu: the weights are N
// gate rows and N up rows. scratch: ta_gemm_mx4_scratch bytes on 16.
#define MX4_MAX_ROWS 64
extern "C" int ta_mx4_max_rows() { return MX4_MAX_ROWS; }
extern "C" int ta_gemm_mx4(hipStream_t stream, int out_dtype, int swiglu, const void* x, long long ldx, const void* codes, const void* scales,
                           const float* bias, void* out, long long ldo, int M, int N, int K, void* scratch, long long scratch_bytes) {
  static const char what[] = "ta_gemm_mx4";
  TA_REQUIRE(out_dtype == TA_F32 || out_dtype == TA_BF16, "%s: unknown dtype %d", what, out_dtype);
  const MxGemm g = {x, nullptr, (const uint8_t*)codes, (const uint8_t*)scales, bias, out, ldx, ldo, M, N, K, out_dtype == TA_F32};
  if (mx_gemm_check(what, g)) return 1;
  TA_REQUIRE(M <= MX4_MAX_ROWS, "%s: %d bfloat16 rows, at most %d", what, M, MX4_MAX_ROWS);
  TA_REQUIRE(ldx >= K && ldx % 8 == 0, "%s: rows %lld apart do not start on 16 bytes", what, ldx);
  // (a tile's rows within 32 bits)
  TA_REQUIRE(ldx <= 1 << 24 && K <= 1 << 23, "%s: rows %lld apart, k %d: at most 16,777,216 and 8,388,608", what, ldx, K);
  TA_REQUIRE(!swiglu || N <= 0x3fffffff, "%s: %d gates", what, N);
  if (M == 0) return 0;
  if (!mx_few(false, swiglu, M, N, K, (uintptr_t)scales % 16 == 0))
    return swiglu ? mx_tiles<false, true>(what, stream, g, scratch, scratch_bytes) : mx_tiles<false, false>(what, stream, g, scratch, scratch_bytes);
  // chunks of 512 where registers allow (1 x 4,096 x 14,336 8.4 us, with 256 8.9); with ups beside the gates 256 (1 x 14,336 x 4,096 15.4, with
  // 512 20.1), as with 16 rows, whose LDS leaves a CU fewer waves (16 x 14,336 x 4,096 14.5 and 17.9). Fewer rows brought: 1 x 4,096 x 14,336
  // with room for 16 12.1
  if (swiglu) {
    if (M <= 1) return mx_few_launch<false, true, 2, 1>(what, stream, g);
    if (M <= 4) return mx_few_launch<false, true, 2, 4>(what, stream, g);
    if (M <= 8) return mx_few_launch<false, true, 2, 8>(what, stream, g);
    return mx_few_launch<false, true, 2, 16>(what, stream, g);
  }
  if (M <= 1) return mx_few_launch<false, false, 4, 1>(what, stream, g);
  if (M <= 4) return mx_few_launch<false, false, 4, 4>(what, stream, g);
  if (mx_few_pairs(false, M, N, K))
    return M <= 8 ? mx_few_launch<false, false, 2, 8, 2>(what, stream, g) : mx_few_launch<false, false, 2, 16, 2>(what, stream, g);
  if (M <= 8) return mx_few_launch<false, false, 4, 8>(what, stream, g);
  return mx_few_launch<false, false, 2, 16>(what, stream, g);
}

static int mx_product8(const char* what, hipStream_t stream, const MxGemm& g, void* scratch, long long scratch_bytes) {
  const int M = g.M, N = g.N, K = g.K;
  if (!mx_few(true, false, M, N, K, ((uintptr_t)g.xs | (uintptr_t)g.scales) % 16 == 0))
    return mx_tiles<true, false>(what, stream, g, scratch, scratch_bytes);
  // (1 x 28,672 x 4,096 in chunks of 512 12.6 us, of 256 14.2; 16 rows 51 and 20.1)
  if (M <= 1) return mx_few_launch<true, false, 4, 1>(what, stream, g);
  if (M <= 4) return mx_few_launch<true, false, 4, 4>(what, stream, g);
  if (mx_few_pairs(true, M, N, K))
    return M <= 8 ? mx_few_launch<true, false, 2, 8, 2>(what, stream, g) : mx_few_launch<true, false, 2, 16, 2>(what, stream, g);
  if (M <= 8) return mx_few_launch<true, false, 2, 8>(what, stream, g);
  return mx_few_launch<true, false, 2, 16>(what, stream, g);
}

// 8-bit rows, codes [M][K] and bytes [M][K/32]; out bfloat16. scratch: ta_gemm_mx4_scratch bytes on 16.
extern "C" int ta_gemm_mx4_mx8(hipStream_t stream, const void* x, const void* xs, const void* codes, const void* scales, const float* bias,
                               void* out, long long ldo, int M, int N, int K, void* scratch, long long scratch_bytes) {
  static const char what[] = "ta_gemm_mx4_mx8";
  const MxGemm g = {x, (const uint8_t*)xs, (const uint8_t*)codes, (const uint8_t*)scales, bias, out, K, ldo, M, N, K, 0};
  if (mx_gemm_check(what, g)) return 1;
  TA_REQUIRE(K <= 1 << 23, "%s: k %d: at most 8,388,608", what, K);         // 256 rows within 31 bits
  if (M > MX_ROWS) {                            // before the first launch: the last may need more than it
    const long long need = ta_gemm_mx4_scratch(1, 0, M, N, K, ((uintptr_t)xs | (uintptr_t)scales) % 16 == 0);
    TA_REQUIRE(need == 0 || (scratch && scratch_bytes >= need && (uintptr_t)scratch % 16 == 0), "%s: %lld bytes of scratch, %lld are needed", what,
               scratch ? scratch_bytes : 0LL, need);
  }
  for (long long at = 0; at < M; at += MX_ROWS) {
    MxGemm part = g;
    part.x = (const uint8_t*)x + at * K;
    part.xs = g.xs + at * (K / MX_BLOCK);
    part.out = (uint8_t*)out + at * ldo * 2;
    part.M = (int)(M - at < MX_ROWS ? M - at : MX_ROWS);
    if (mx_product8(what, stream, part, scratch, scratch_bytes)) return 1;
  }
  return 0;
}
