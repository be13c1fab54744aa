// To and from the blocks of mx.h: matrices to 4-bit weights and back, rows to 8 bits, and the two kernels that leave rows in
// 8 bits where a step forms them: the norm behind the residual's addition, and the gated activation. All are bound by
// memory: a lane takes 8 neighbouring values, the quad of its neighbours a block, so that the largest magnitude takes
// two exchanges inside the quad. Pieces of 8 are counted in 32 bits (a division in 64 is some 150 instructions a lane); a
// launch holds rows of 2^31 of them at most, more rows are several launches.
#include "mx.h"

// ------------------------------------------------------------------ matrices
// w [n][k] -> codes [n][k/2], scales [n][k/32]; a thread takes 8 values
template <typename T>
__global__ __launch_bounds__(256) void mx4_pack_kernel(const T* __restrict__ w, long long ldw, uint8_t* __restrict__ codes,
                                                       uint8_t* __restrict__ scales, uint32_t n, int k) {
  const uint32_t pieces = k / 8, at = blockIdx.x * 256 + threadIdx.x;
  const bool ok = at < n * pieces;               // a block's four threads are in or out together
  const long long row = ok ? at / pieces : 0, p = ok ? at % pieces : 0;
  float v[8];
  mx_load8(w + row * ldw + p * 8, v);
  const uint32_t byte = mx4_scale_byte(mx_top_quad(mx_top8(v)));
  if (!ok) return;
  uint32_t c = 0;
  if (byte != MX_NAN) {
    const float s = mx_inverse(byte);
#pragma unroll
    for (int i = 0; i < 8; ++i) c |= mx4_code(v[i] * s) << (4 * i);
  }
  *reinterpret_cast<uint32_t*>(codes + row * (k / 2) + p * 4) = c;
  if (p % 4 == 0) scales[row * (k / 32) + p / 4] = (uint8_t)byte;
}

// the values that the codes stand for, exactly (bfloat16 holds them all but those below 2^-133 or above its range)
template <typename T>
__global__ __launch_bounds__(256) void mx4_unpack_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                         T* __restrict__ out, long long ldo, uint32_t n, int k) {
  const uint32_t pieces = k / 8, at = blockIdx.x * 256 + threadIdx.x;
  if (at >= n * pieces) return;
  const long long row = at / pieces, p = at % pieces;
  const uint32_t c = *reinterpret_cast<const uint32_t*>(codes + row * (k / 2) + p * 4);
  const float s = mx_scale(scales[row * (k / 32) + p / 4]);
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t m = c >> (4 * i) & 7u, sign = c >> (4 * i + 3) & 1u;
    // exponent field 0: m / 2; else (1 + last bit / 2) 2^(field - 1)
    const float a = m < 2 ? 0.5f * (float)m : __uint_as_float(((m >> 1) + 126u) << 23 | (m & 1u) << 22);
    v[i] = (sign ? -a : a) * s;
  }
  T* o = out + row * ldo + p * 8;
  if (sizeof(T) == 2) {
    mx_u32x4 q;
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = f32x2_to_bf16x2_bits(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<mx_u32x4*>(o) = q;
  } else {
    reinterpret_cast<float4*>(o)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(o)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}

static bool mx_on(const void* p, int bytes) { return (uintptr_t)p % (uintptr_t)bytes == 0; }
static int mx_blocks(const char* what, long long n, int k) {
  TA_REQUIRE(n >= 0 && k >= MX_BLOCK && k % MX_BLOCK == 0, "%s: %lld rows of %d: k goes by blocks of %d", what, n, k, MX_BLOCK);
  return 0;
}
// launch(first row, rows, workgroups) for as many rows at a time as 2^31 pieces are
template <typename F>
static int mx_rows_launch(const char* what, long long n, int k, F launch) {
  const long long most = (1LL << 31) / (k / 8);
  for (long long at = 0; at < n; at += most) {
    const long long rows = n - at < most ? n - at : most;
    launch(at, (uint32_t)rows, (unsigned)((rows * (k / 8) + 255) / 256));
    if (ta_check_launch(what)) return 1;
  }
  return 0;
}

// w [n][ldw] float32 or bfloat16, rows on 16 bytes.
extern "C" int ta_mx4_pack(hipStream_t stream, int dtype, const void* w, long long ldw, void* codes, void* scales, long long n, int k) {
  TA_REQUIRE(dtype == TA_F32 || dtype == TA_BF16, "ta_mx4_pack: unknown dtype %d", dtype);
  if (mx_blocks("ta_mx4_pack", n, k)) return 1;
  TA_REQUIRE(ldw >= k && ldw * (dtype == TA_F32 ? 4 : 2) % 16 == 0 && mx_on(w, 16) && mx_on(codes, 16),
             "ta_mx4_pack: rows %lld apart do not start on 16 bytes", ldw);
  return mx_rows_launch("ta_mx4_pack", n, k, [&](long long at, uint32_t rows, unsigned grid) {
    uint8_t *c = (uint8_t*)codes + at * (k / 2), *s = (uint8_t*)scales + at * (k / 32);
    if (dtype == TA_F32) mx4_pack_kernel<float><<<grid, 256, 0, stream>>>((const float*)w + at * ldw, ldw, c, s, rows, k);
    else mx4_pack_kernel<bf16_t><<<grid, 256, 0, stream>>>((const bf16_t*)w + at * ldw, ldw, c, s, rows, k);
  });
}

extern "C" int ta_mx4_unpack(hipStream_t stream, int dtype, const void* codes, const void* scales, void* out, long long ldo, long long n,
                             int k) {
  TA_REQUIRE(dtype == TA_F32 || dtype == TA_BF16, "ta_mx4_unpack: unknown dtype %d", dtype);
  if (mx_blocks("ta_mx4_unpack", n, k)) return 1;
  TA_REQUIRE(ldo >= k && ldo * (dtype == TA_F32 ? 4 : 2) % 16 == 0 && mx_on(out, 16) && mx_on(codes, 16),
             "ta_mx4_unpack: rows %lld apart do not start on 16 bytes", ldo);
  return mx_rows_launch("ta_mx4_unpack", n, k, [&](long long at, uint32_t rows, unsigned grid) {
    const uint8_t *c = (const uint8_t*)codes + at * (k / 2), *s = (const uint8_t*)scales + at * (k / 32);
    if (dtype == TA_F32) mx4_unpack_kernel<float><<<grid, 256, 0, stream>>>(c, s, (float*)out + at * ldo, ldo, rows, k);
    else mx4_unpack_kernel<bf16_t><<<grid, 256, 0, stream>>>(c, s, (bf16_t*)out + at * ldo, ldo, rows, k);
  });
}

// ------------------------------------------------------------------ rows
template <typename T>
__global__ __launch_bounds__(256) void mx8_pack_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ codes,
                                                       uint8_t* __restrict__ scales, uint32_t n, int k) {
  const uint32_t pieces = k / 8, at = blockIdx.x * 256 + threadIdx.x;
  if (at >= n * pieces) return;                  // a block's four threads are in or out together
  const long long row = at / pieces, p = at % pieces;
  float v[8];
  mx_load8(x + row * ldx + p * 8, v);
  mx8_store(v, codes + row * k + p * 8, scales + row * (k / 32) + p / 4);
}

extern "C" int ta_mx8_pack(hipStream_t stream, int dtype, const void* x, long long ldx, void* codes, void* scales, long long n, int k) {
  TA_REQUIRE(dtype == TA_F32 || dtype == TA_BF16, "ta_mx8_pack: unknown dtype %d", dtype);
  if (mx_blocks("ta_mx8_pack", n, k)) return 1;
  TA_REQUIRE(ldx >= k && ldx * (dtype == TA_F32 ? 4 : 2) % 16 == 0 && mx_on(x, 16) && mx_on(codes, 16),
             "ta_mx8_pack: rows %lld apart do not start on 16 bytes", ldx);
  return mx_rows_launch("ta_mx8_pack", n, k, [&](long long at, uint32_t rows, unsigned grid) {
    uint8_t *c = (uint8_t*)codes + at * k, *s = (uint8_t*)scales + at * (k / 32);
    if (dtype == TA_F32) mx8_pack_kernel<float><<<grid, 256, 0, stream>>>((const float*)x + at * ldx, ldx, c, s, rows, k);
    else mx8_pack_kernel<bf16_t><<<grid, 256, 0, stream>>>((const bf16_t*)x + at * ldx, ldx, c, s, rows, k);
  });
}

// g / (1 + exp(-g)) within about a unit of its last bit, for |g| <= 80: exp2 of the rounded exponent times what the rounding
// left out, and a quotient with one step behind the hardware's reciprocal. With the library's exponential and a
// full division, which ask about ranges that no gate here has, 4,096 x 14,336 took 66 us, bound by instructions and not by memory.
__device__ __forceinline__ float mx_silu(float g) {
  constexpr float L = 1.44269502f, L_REST = 1.92596303e-8f, LN2 = 0.693147182f;       // log2(e) = L + L_REST
  const float t = -g * L, rest = fmaf(-g, L_REST, fmaf(-g, L, -t));
  const float e = __builtin_amdgcn_exp2f(t), d = 1.0f + fmaf(e, rest * LN2, e);
  const float y = __builtin_amdgcn_rcpf(d), s = g * y;
  return fmaf(fmaf(-d, s, g), y, s);
}

// silu(gate) * up of [gate | up] rows, to 8 bits. The error is that of 32-bit arithmetic: a value next to a rounding border of
// e4m3 falls where that puts it.
template <typename T>
__global__ __launch_bounds__(256) void swiglu_mx8_kernel(const T* __restrict__ gu, long long ld, const float* __restrict__ bias,
                                                         uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, uint32_t n, int d) {
  const uint32_t pieces = d / 8, at = blockIdx.x * 256 + threadIdx.x;
  if (at >= n * pieces) return;
  const long long row = at / pieces;
  const int p = (int)(at % pieces);
  float g[8], u[8];
  mx_load8(gu + row * ld + p * 8, g);
  mx_load8(gu + row * ld + d + p * 8, u);
  if (bias) {
    float bg[8], bu[8];
    mx_load8(bias + p * 8, bg);
    mx_load8(bias + d + p * 8, bu);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      g[i] += bg[i];
      u[i] += bu[i];
    }
  }
  // a gate beyond 80 (NaN and infinities have bits above it too) goes by the library's functions, itself alone: a value's bits are its own
  // gate's and up's, whatever else its row or its wave holds
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = mx_silu(g[i]);
  if (mx_top8(g) > 0x42a00000u) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((__float_as_uint(g[i]) & 0x7fffffffu) > 0x42a00000u) y[i] = g[i] / (1.0f + expf(-g[i]));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] *= u[i];
  mx8_store(y, codes + row * d + p * 8, scales + row * (d / 32) + p / 4);
}

// gate_up [n][ld] float32 or bfloat16: d gates, then d ups; bias [2 d] or null.
extern "C" int ta_swiglu_mx8(hipStream_t stream, int dtype, const void* gate_up, long long ld, const float* bias, void* codes, void* scales,
                             long long n, int d) {
  TA_REQUIRE(dtype == TA_F32 || dtype == TA_BF16, "ta_swiglu_mx8: unknown dtype %d", dtype);
  if (mx_blocks("ta_swiglu_mx8", n, d)) return 1;
  TA_REQUIRE(ld >= 2LL * d && ld * (dtype == TA_F32 ? 4 : 2) % 16 == 0 && mx_on(gate_up, 16) && mx_on(codes, 16) && mx_on(bias, 16),
             "ta_swiglu_mx8: rows %lld apart do not start on 16 bytes", ld);
  return mx_rows_launch("ta_swiglu_mx8", n, d, [&](long long at, uint32_t rows, unsigned grid) {
    uint8_t *c = (uint8_t*)codes + at * d, *s = (uint8_t*)scales + at * (d / 32);
    if (dtype == TA_F32) swiglu_mx8_kernel<float><<<grid, 256, 0, stream>>>((const float*)gate_up + at * ld, ld, bias, c, s, rows, d);
    else swiglu_mx8_kernel<bf16_t><<<grid, 256, 0, stream>>>((const bf16_t*)gate_up + at * ld, ld, bias, c, s, rows, d);
  });
}

// ------------------------------------------------------------------ add + norm
// v = x + delta (+ bias), stored to `stream` where there is one; y = v / sqrt(mean(v^2) + eps) * weight, to 8 bits. One
// workgroup a row; HELD pieces of 8 values a thread stay in registers between the sum and the rows, 0: any number, read again
// (by the thread that stored them).
//
// What becomes the rows is added and normed in 64 bits beside the stream's 32 and rounded once, to e4m3: an error of 2^-24 moves one
// in some 10^6 values over the middle between two codes, a sixteenth of itself away, and that would be the largest error there is.
// It costs 3 of 42 us (2,048 rows of 8,192 with a bias: conversions, a quarter of the rate). Without registers for a row's pieces the
// norm goes by the stream's values.
__device__ __forceinline__ double mx_sum64(double v) {
  const auto take = [&](auto ctrl) {
    const mx_u32x2 b = __builtin_bit_cast(mx_u32x2, v);
    v += __builtin_bit_cast(double, mx_u32x2{(uint32_t)__builtin_amdgcn_update_dpp(0, (int)b[0], decltype(ctrl)::value, 0xf, 0xf, true),
                                             (uint32_t)__builtin_amdgcn_update_dpp(0, (int)b[1], decltype(ctrl)::value, 0xf, 0xf, true)});
  };
  take(std::integral_constant<int, 0xb1>());     // pairs, quads, halves of a row, rows
  take(std::integral_constant<int, 0x4e>());
  take(std::integral_constant<int, 0x141>());
  take(std::integral_constant<int, 0x140>());
  const mx_u32x2 b = __builtin_bit_cast(mx_u32x2, v);
  double rows[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    rows[i] = __builtin_bit_cast(double, mx_u32x2{(uint32_t)__builtin_amdgcn_readlane((int)b[0], 16 * i),
                                                  (uint32_t)__builtin_amdgcn_readlane((int)b[1], 16 * i)});
  return (rows[0] + rows[1]) + (rows[2] + rows[3]);
}

// to 32 bits by truncation with the last bit set where anything is lost: a rounding to fewer bits then goes as from y itself
__device__ __forceinline__ float mx_odd(double y) {
  const float near = (float)y;
  const double back = near;
  uint32_t bits = __float_as_uint(near);
  bits -= fabs(back) > fabs(y) && !isinf(near);
  bits |= back != y && !isinf(near);
  return __uint_as_float(bits);
}

template <typename TD, int THREADS, int HELD>
__global__ __launch_bounds__(THREADS) void add_rmsnorm_mx8_kernel(const float* x, const TD* __restrict__ delta,
                                                                  long long plane, int planes, const float* __restrict__ bias,
                                                                  const float* __restrict__ weight, float eps, float* to,
                                                                  uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int d, double share) {
  const size_t base = (size_t)blockIdx.x * d;
  const int pieces = d / 8;
  __shared__ double part[THREADS / 64];
  double held[HELD ? HELD : 1][8];
  double sum = 0.;
  const auto form = [&](int p, double* wide) {
    float v[8];
    mx_load8(x + base + p * 8, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) wide[i] = v[i];
    const auto add = [&](const float* t) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] += t[i];
        wide[i] += t[i];
      }
    };
    for (int j = 0; j < planes; ++j) {
      float t[8];
      mx_load8(delta + j * plane + base + p * 8, t);
      add(t);
    }
    if (bias) {
      float t[8];
      mx_load8(bias + p * 8, t);
      add(t);
    }
    if (to) {
      reinterpret_cast<float4*>(to + base + p * 8)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(to + base + p * 8)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (!HELD) wide[i] = v[i];
      sum += wide[i] * wide[i];
    }
  };
  if (HELD) {
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
      const int p = threadIdx.x + h * THREADS;
      if (p < pieces) form(p, held[h]);
    }
  } else {
    for (int p = threadIdx.x; p < pieces; p += THREADS) form(p, held[0]);
  }
  sum = mx_sum64(sum);
  if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = sum;
  __syncthreads();
  double all = 0.;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) all += part[w];
  // the unit's root, good to some 26 bits, and a step of Newton's; 0 and infinity stay as they are
  const double mean = all * share + (double)eps, near = __builtin_amdgcn_rsq(mean), better = near * (1.5 - 0.5 * mean * near * near);
  const double r = isnan(better) ? near : better;
  const auto leave = [&](int p, const double* v) {
    float w[8], y[8];
    mx_load8(weight + p * 8, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = mx_odd(v[i] * r * w[i]);
    mx8_store(y, codes + base + p * 8, scales + base / 32 + p / 4);
  };
  if (HELD) {
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
      const int p = threadIdx.x + h * THREADS;
      if (p < pieces) leave(p, held[h]);
    }
  } else {
    const float* from = to ? to : x;
    for (int p = threadIdx.x; p < pieces; p += THREADS) {
      float v[8];
      mx_load8(from + base + p * 8, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) held[0][i] = v[i];
      leave(p, held[0]);
    }
  }
}

template <typename TD>
static void launch_norm(hipStream_t stream, const float* x, const TD* delta, int planes, const float* bias, const float* weight, float eps,
                        float* to, uint8_t* codes, uint8_t* scales, int n, int d, long long plane) {
#define MX_NORM(T, H) add_rmsnorm_mx8_kernel<TD, T, H><<<n, T, 0, stream>>>(x, delta, plane, planes, bias, weight, eps, to, codes, scales, d, 1. / d)
  // as many threads as a row has pieces: out of memory 8 x 8,192 4.1 us (with 512 threads of two pieces 5.2), 2,048 x 8,192 42.3 (42.9), 2,048 x
  // 4,096 22.1 (with 256 threads of two 23.0)
  if (d <= 2048) MX_NORM(256, 1);
  else if (d <= 4096) MX_NORM(512, 1);
  else if (d <= 8192) MX_NORM(1024, 1);
  else if (d <= 16384) MX_NORM(1024, 2);
  else if (d <= 32768) MX_NORM(1024, 4);
  else MX_NORM(1024, 0);
#undef MX_NORM
}

// x [n][d] float32; delta: null (planes 0), or planes of [n][d], float32 or bfloat16, added in order; bias [d] or null; to: null, x,
// or another [n][d] that gets the sum.
extern "C" int ta_add_rmsnorm_mx8(hipStream_t stream, int delta_dtype, const float* x, const void* delta, int planes, const float* bias,
                                  const float* weight, float eps, float* to, void* codes, void* scales, int n, int d) {
  TA_REQUIRE(delta_dtype == TA_F32 || delta_dtype == TA_BF16, "ta_add_rmsnorm_mx8: unknown dtype %d", delta_dtype);
  TA_REQUIRE(n >= 0 && d >= MX_BLOCK && d % MX_BLOCK == 0, "ta_add_rmsnorm_mx8: %d rows of %d: rows go by blocks of %d", n, d, MX_BLOCK);
  TA_REQUIRE(planes >= 0 && planes <= TA_MAX_PLANES && (planes > 0) == (delta != nullptr), "ta_add_rmsnorm_mx8: %d planes", planes);
  TA_REQUIRE(mx_on(x, 16) && mx_on(delta, 16) && mx_on(bias, 16) && mx_on(weight, 16) && mx_on(to, 16) && mx_on(codes, 16),
             "ta_add_rmsnorm_mx8: rows do not start on 16 bytes");
  TA_REQUIRE(to || (planes == 0 && !bias), "ta_add_rmsnorm_mx8: what is added goes nowhere");
  // a launch has fewer than 2^32 threads, and a row has up to 1,024 of them
  const long long most = 1 << 21, plane = (long long)n * d;
  for (long long at = 0; at < n; at += most) {
    const int rows = (int)(n - at < most ? n - at : most);
    const long long from = at * d;
    uint8_t *c = (uint8_t*)codes + from, *s = (uint8_t*)scales + from / MX_BLOCK;
    float* sum = to ? to + from : nullptr;
    if (delta_dtype == TA_F32)
      launch_norm<float>(stream, x + from, delta ? (const float*)delta + from : nullptr, planes, bias, weight, eps, sum, c, s, rows, d, plane);
    else
      launch_norm<bf16_t>(stream, x + from, delta ? (const bf16_t*)delta + from : nullptr, planes, bias, weight, eps, sum, c, s, rows, d, plane);
    if (ta_check_launch("ta_add_rmsnorm_mx8")) return 1;
  }
  return 0;
}
