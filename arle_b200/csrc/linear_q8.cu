// Activations and weights as e4m3 codes (q8.cuh), for the products of gemm_q8.cu.
//
// Rows: numbers of k are taken in groups of 128 (kb = ceil(K / 128) of them; the last is filled up with codes of zero).  A group's scale is the least
// power of two s with max |x| <= 448 s (2^-100 to 2^119), stored as its exponent (e8m0: exponent + 127); codes are rne(x / s).  Numbers that are not
// finite do not count for the scale and become NaN: e4m3 has no infinities, and what was not finite must not come out of a product as if it were.
// Weights: the same for blocks of 128 x 128, one float32 scale a block.
// All are launched early: plain loads, and what a block loads is small beside what its neighbours have under way.  It saves one token's codes 0.4 us in a
// chain, a weight of 24,576 x 4,096 2, the norm of 1,024 rows of 4,096 0.4 and that of 4,096 rows 0.9 (a weight's kernel lets nothing start before its end: it runs once, at load).
// The kernels read a number once and keep it in registers between the maximum and the rounding (twice: norms whose rows are not on 16-byte boundaries or too long to keep,
// weights with numbers that are not finite, rows of extreme_row), and are bound by DRAM (few rows: by latency).  Times are those of a kernel alone in a captured graph.
#include "q8.cuh"
#include "scan_utils.cuh"
using namespace arle;

namespace {

constexpr int kGroup = 128;

// The maximum of `bits` over the 2^k lanes that share lane / LANES.
template <int LANES> __device__ __forceinline__ uint32_t lanes_max(uint32_t bits) {
  if constexpr (LANES == 32) {
    return __reduce_max_sync(0xffffffffu, bits);
  } else {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
    return bits;
  }
}

// The codes of a group that LANES lanes hold, V consecutive numbers each, from the bits of its largest: returns the scale, words of four codes in `w`.
template <int LANES, int V> __device__ __forceinline__ float group_codes(float (&v)[V], uint32_t (&w)[V / 4], uint32_t most) {
  if (LANES == 32 ? most >= kInfBits : __any_sync(0xffffffffu, most >= kInfBits) != 0) {
    most = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) most = max(most, finite_bits(v[j])), v[j] = finite_or_nan(v[j]);
    most = lanes_max<LANES>(most);
  }
  const float s = q8_scale(__uint_as_float(most)), inv = inverse_scale(s);
#pragma unroll
  for (int j = 0; j < V / 4; ++j) w[j] = q8_codes4(v[4 * j] * inv, v[4 * j + 1] * inv, v[4 * j + 2] * inv, v[4 * j + 3] * inv);
  return s;
}

template <int LANES, int V> __device__ __forceinline__ float group_codes(float (&v)[V], uint32_t (&w)[V / 4]) {
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) most = max(most, abs_bits(v[j]));
  return group_codes<LANES, V>(v, w, lanes_max<LANES>(most));
}

// 16 bytes of a row as they lie in memory, of which `left` numbers are there (the others are zero), and their largest without its sign: bfloat16 numbers two at a
// time, `fold` brings the two together as the bits of a float32 number.
template <typename T, bool ALIGNED> __device__ __forceinline__ uint4 load_words(const T* p, int left) {
  if constexpr (ALIGNED) {
    return left > 0 ? *reinterpret_cast<const uint4*>(p) : make_uint4(0u, 0u, 0u, 0u);
  } else {
    constexpr int V = 16 / sizeof(T);
    Pack<T, V> e;
#pragma unroll
    for (int j = 0; j < V; ++j) e.e[j] = j < left ? p[j] : from_f32<T>(0.f);
    return *reinterpret_cast<const uint4*>(&e);
  }
}
template <typename T> __device__ __forceinline__ uint32_t largest(uint32_t a, uint32_t b) { return sizeof(T) == 2 ? __vmaxu2(a, b) : max(a, b); }
template <typename T> __device__ __forceinline__ uint32_t largest(uint4 q) {
  constexpr uint32_t magnitude = sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu;
  return largest<T>(largest<T>(q.x & magnitude, q.y & magnitude), largest<T>(q.z & magnitude, q.w & magnitude));
}
template <typename T> __device__ __forceinline__ uint32_t fold(uint32_t m) { return sizeof(T) == 2 ? max(m << 16, m & 0xffff0000u) : m; }

// V numbers from p on, of which `left` are there (the others are zero).
template <typename T, int V, bool ALIGNED> __device__ __forceinline__ void load_numbers(const T* p, int left, float (&v)[V]) {
  if constexpr (ALIGNED) {
    if (left >= V) {
      load_vec<T, V>(p, v);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = 0.f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = j < left ? to_f32(p[j]) : 0.f;
  }
}

// ------------------------------------------------------------------ rows
// A lane takes 16 bytes of a group: a group is 16 lanes of bfloat16 or 32 of float32; it takes them of kAtOnce groups, which are under way together (one at a time
// 6,001 rows of 8,192 bfloat16 took 37 us, four 28), and stay as they lie in memory up to the rounding: maxima of two bfloat16 at a time, and a multiplication for
// the division by the row's groups, 23.6: 6.4 TB/s (26.6 among calls from Python one by one).  One row of 4,096 1.6 us.
constexpr int kAtOnce = 4;

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* x, long row_stride, uint8_t* codes, uint8_t* scales, uint32_t groups, int K, uint32_t kb, uint32_t magic,
                                                            int shift) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int V = 16 / sizeof(T), LANES = kGroup / V, GROUPS = 256 / LANES;
  const int sub = threadIdx.x % LANES;
  const uint32_t g0 = blockIdx.x * (GROUPS * kAtOnce) + threadIdx.x / LANES;
  uint4 kept[kAtOnce];
#pragma unroll
  for (int u = 0; u < kAtOnce; ++u) {
    const uint32_t g = g0 + u * GROUPS, row = __umulhi(2u * g, magic) >> shift;      // g / kb
    const int at = (int)(g - row * kb) * kGroup + sub * V;
    kept[u] = load_words<T, ALIGNED>(x + (long)(g < groups ? row : 0) * row_stride + at, g < groups ? K - at : 0);
  }
#pragma unroll
  for (int u = 0; u < kAtOnce; ++u) {
    const uint32_t g = g0 + u * GROUPS;
    const Pack<T, V> p = *reinterpret_cast<const Pack<T, V>*>(&kept[u]);
    uint32_t most = largest<T>(kept[u]), w[V / 4];
    if constexpr (LANES == 32) {
      most = __reduce_max_sync(0xffffffffu, most);
    } else {
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) most = largest<T>(most, __shfl_xor_sync(0xffffffffu, most, o));
    }
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = to_f32(p.e[j]);
    const float s = group_codes<LANES, V>(v, w, fold<T>(most));
    if (g >= groups) continue;
    uint8_t* dst = codes + (size_t)g * kGroup + sub * V;
    if constexpr (V == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(dst) = w[0];
    if (sub == 0) scales[g] = exponent_byte(s);
  }
}

// ------------------------------------------------------------------ weights
// A block of 256 threads owns 128 x 128 numbers, which are all under way at once and stay as they lie in memory between the maximum and the rounding.  Where a
// number is not finite they are read again.  24,576 x 4,096 bfloat16 45 us, 6.7 TB/s; 1,001 x 777 float32, whose rows are not aligned, 3.3 us (6.4 when they were read twice).
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256, ALIGNED && sizeof(T) == 2 ? 4 : 2) quantize_weight_kernel(const T* w, long row_stride, uint8_t* codes, float* scales, int N, int K, int kb) {
  pdl_wait();
  constexpr int V = 16 / sizeof(T), LANES = kGroup / V, ROWS = 256 / LANES, STEPS = kGroup / ROWS;
  __shared__ uint32_t most_s[8];
  const int b = blockIdx.x, sub = threadIdx.x % LANES, n0 = blockIdx.y * kGroup + threadIdx.x / LANES, at = b * kGroup + sub * V;
  uint8_t* dst = codes + (size_t)n0 * kb * kGroup + at;
  const size_t step = (size_t)ROWS * kb * kGroup;
  auto block_max = [&](uint32_t most) {
    most = lanes_max<32>(most);
    if ((threadIdx.x & 31) == 0) most_s[threadIdx.x >> 5] = most;
    __syncthreads();
    most = most_s[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) most = max(most, most_s[i]);
    return most;
  };
  auto put = [&](int i, const float (&v)[V], float inv) {
    uint32_t c[V / 4];
#pragma unroll
    for (int j = 0; j < V / 4; ++j) c[j] = q8_codes4(v[4 * j] * inv, v[4 * j + 1] * inv, v[4 * j + 2] * inv, v[4 * j + 3] * inv);
    if constexpr (V == 8) *reinterpret_cast<uint2*>(dst + i * step) = make_uint2(c[0], c[1]);
    else *reinterpret_cast<uint32_t*>(dst + i * step) = c[0];
  };
  {
    uint4 kept[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int n = n0 + i * ROWS;
      kept[i] = load_words<T, ALIGNED>(w + (long)n * row_stride + at, n < N ? K - at : 0);
    }
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) most = largest<T>(most, largest<T>(kept[i]));
    most = block_max(fold<T>(most));
    if (most < kInfBits) {
      const float s = q8_scale(__uint_as_float(most)), inv = inverse_scale(s);
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        if (n0 + i * ROWS >= N) break;
        const Pack<T, V> p = *reinterpret_cast<const Pack<T, V>*>(&kept[i]);
        float v[V];
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = to_f32(p.e[j]);
        put(i, v, inv);
      }
      if (threadIdx.x == 0) scales[(size_t)blockIdx.y * kb + b] = s;
      return;
    }
    __syncthreads();                                       // the maxima have been read
  }
  auto numbers = [&](int i, float (&v)[V]) {
    const int n = n0 + i * ROWS;
    load_numbers<T, V, false>(w + (long)(n < N ? n : 0) * row_stride + at, n < N ? K - at : 0, v);
  };
  uint32_t most = 0;
#pragma unroll 2
  for (int i = 0; i < STEPS; ++i) {
    float v[V];
    numbers(i, v);
#pragma unroll
    for (int j = 0; j < V; ++j) most = max(most, finite_bits(v[j]));
  }
  const float s = q8_scale(__uint_as_float(block_max(most))), inv = inverse_scale(s);
#pragma unroll 2
  for (int i = 0; i < STEPS; ++i) {
    if (n0 + i * ROWS >= N) break;
    float v[V];
    numbers(i, v);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = finite_or_nan(v[j]);
    put(i, v, inv);
  }
  if (threadIdx.x == 0) scales[(size_t)blockIdx.y * kb + b] = s;
}

// The block's sum of its warps' sums, the same in every thread; blocks of whole warps, up to 32 of them.
__device__ __forceinline__ double block_sum64(double s, double* scratch) {
  if (blockDim.x == 32) return s;
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = s;
  __syncthreads();
  s = (threadIdx.x & 31) < (blockDim.x >> 5) ? scratch[threadIdx.x & 31] : 0.0;
  if (blockDim.x > 512) s += __shfl_xor_sync(0xffffffffu, s, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return __shfl_sync(0xffffffffu, s, 0);                    // (lanes from 16 on have added zeros only)
}

// Two differences a - b, rounded towards zero, the last bit set where that left something out: a number that lies beside a border between two codes (or
// two scales), which have zeros there, stays on its side of it, as if nothing had been rounded.
__device__ __forceinline__ void subtract_sticky(f32x2 a, f32x2 b, float& lo, float& hi) {
  f32x2 s, back;
  asm("sub.rz.f32x2 %0, %1, %2;" : "=l"(s) : "l"(a), "l"(b));
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(back) : "l"(a), "l"(s));            // b where s is a - b, with no rounding of its own (|b| is far below |a|)
  lo = low2(back) != low2(b) ? __uint_as_float(__float_as_uint(low2(s)) | 1u) : low2(s);
  hi = high2(back) != high2(b) ? __uint_as_float(__float_as_uint(high2(s)) | 1u) : high2(s);
}

// 1 / sqrt(m) as two float32 numbers: an approximation y and half its residual, y + y (1 - m y^2) / 2 (one step of Newton's method).  For m in kLeastMean .. kMostMean,
// where y^2, its rounding error and what m has beside its float32 number are all normal numbers, and the sums of squares behind m are.
constexpr float kLeastMean = 0x1p-90f, kMostMean = 0x1p100f;
__device__ __forceinline__ float2 inverse_root(double m) {
  const float mh = (float)m, ml = (float)(m - (double)mh), y = rsqrtf(mh);
  const float q = y * y, ql = fmaf(y, y, -q);
  const float r = fmaf(-mh, q, 1.0f) - fmaf(mh, ql, ml * q);
  return make_float2(y, 0.5f * y * r);
}

// ------------------------------------------------------------------ residual sum, norm, codes
// A code is off where an error carries a number over the border between two codes, in steps of an eighth of the number.  So the sum of squares is of 64 bits from a
// warp's sums on, the factor of a row is a pair of float32 numbers, and where its product with a number would round onto a border it is rounded as subtract_sticky
// does.  Of the 25.6 million codes of 5,003 rows of 5,120, 17 are off in a careful float32 form, 14 with products rounded to float32, three so (54.0 and 55.6 us when that
// was chosen; four and 56.9 with every product rounded so).
struct RowFactor { f32x2 hi, lo, minus_hi, minus_lo; };       // each twice

__device__ __forceinline__ void finish_four(float (&v)[4], const float (&g)[4], const RowFactor& r, uint8_t* codes, uint8_t* scales, size_t first_group, int slot) {
  uint32_t w[1];
  f32x2 ys[2], rests[2];
#pragma unroll
  for (int j = 0; j < 4; j += 2) {                          // v (hi + lo) g, to some 2^-45 (not finite: NaN)
    const f32x2 v2 = pair2(v[j], v[j + 1]), g2 = pair2(g[j], g[j + 1]);
    const f32x2 f = mul2(r.hi, g2), minus_f = mul2(r.minus_hi, g2), y = mul2(v2, f);
    const f32x2 minus_fl = fma2(r.minus_lo, g2, fma2(r.minus_hi, g2, f));           // what f lacks, with its sign turned
    const f32x2 minus_rest = fma2(v2, minus_fl, fma2(v2, minus_f, y));
    ys[j / 2] = y, rests[j / 2] = minus_rest;
    v[j] = low2(y) - low2(minus_rest), v[j + 1] = high2(y) - high2(minus_rest);
  }
  // (the borders' last 19 bits are zeros: four bits say which code, or half a step more)
  auto low_bits = [](float a) { return __float_as_uint(a) & 0x7ffffu; };
  if (min(min(low_bits(v[0]), low_bits(v[1])), min(low_bits(v[2]), low_bits(v[3]))) == 0) {
    subtract_sticky(ys[0], rests[0], v[0], v[1]);
    subtract_sticky(ys[1], rests[1], v[2], v[3]);
  }
  const float s = group_codes<32, 4>(v, w);
  const size_t group = first_group + (slot >> 5);
  *reinterpret_cast<uint32_t*>(codes + group * kGroup + 4 * (slot & 31)) = w[0];
  if ((slot & 31) == 0) scales[group] = exponent_byte(s);
}

// A row whose mean square float32 does not carry: numbers whose squares leave its range (from some 10^15 on, or below 10^-13 beside no eps), infinities
// (they come out as NaN and the row's finite numbers as zero, 1 / sqrt(inf) times them), NaN (all of the row).  Everything in 64 bits, from the numbers in memory:
// `x` and, where their sum is kept nowhere, `delta`.  The filled-up columns are zero whatever the row holds.  It comes behind the others' path and writes over what
// that made, each thread its own places: a branch in the middle, around which the compiler moves nothing, made all rows slower (5,003 rows of 5,120, alone in a graph,
// 57.5 us; at the end 56.6; with no second path 55.5).
template <typename TA>
__device__ __noinline__ void extreme_row(const float* x, const TA* delta, float delta_scale, const float* gain, uint8_t* codes, uint8_t* scales, int H, int kb,
                                         double inv_h, float eps, double* scratch) {
  auto number = [&](int at) { return at >= H ? 0.f : delta ? fmaf(delta_scale, to_f32(delta[at]), x[at]) : x[at]; };
  double ss = 0.0;
  for (int slot = threadIdx.x; slot < 32 * kb; slot += blockDim.x)
    for (int j = 0; j < 4; ++j) {
      const double v = number(4 * slot + j);
      ss += v * v;
    }
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  __syncthreads();                                          // the scratch has been read
  const double r = 1.0 / sqrt(block_sum64(ss, scratch) * inv_h + (double)eps);
  for (int slot = threadIdx.x; slot < 32 * kb; slot += blockDim.x) {
    float v[4];
    for (int j = 0; j < 4; ++j) {
      const int at = 4 * slot + j;
      const double y = at < H ? (double)number(at) * r * (double)gain[at] : 0.0;
      v[j] = __double2float_rz(y);                          // the last bit set where that left something out (see subtract_sticky)
      if ((double)v[j] != y) v[j] = __uint_as_float(__float_as_uint(v[j]) | 1u);
    }
    uint32_t w[1];
    const float s = group_codes<32, 4>(v, w);
    *reinterpret_cast<uint32_t*>(codes + 4 * (size_t)slot) = w[0];
    if ((slot & 31) == 0) scales[slot >> 5] = exponent_byte(s);
  }
}

// One block a row; a warp and step hold one group.  PER > 0: a thread keeps PER float4 of the row (rows on 16-byte boundaries); PER = 0: the row is
// read twice, number by number.  5,003 rows of 5,120 56.6 us, 5.0 TB/s, 60 among calls from Python one by one (4 more with half the warps on an SM, 65 with blocks that stay and copy the next row to shared
// memory meanwhile): reads, a sum over the block and writes of a row follow one another, and what hides that is other rows' warps.  Eight rows of 4,096 2.5 us alone.
template <typename TA, int PER>
__global__ void __launch_bounds__(1024, PER == 4 ? 1 : 2) rmsnorm_q8_kernel(const float* resid, const TA* delta, const float* gain, float* sum_out, uint8_t* codes,
                                                          uint8_t* scales, int H, int kb, double inv_h, float eps, float delta_scale) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ double red[32];
  constexpr int KEEP = PER > 0 ? PER : 1;
  const long row = blockIdx.x;
  const float* xr = resid + row * H;
  const TA* dr = delta ? delta + row * H : nullptr;
  float* so = sum_out ? sum_out + row * H : nullptr;
  const int slots = kb * 32;                                // of four numbers
  f32x2 ss = 0;                                             // two sums, of even and odd places
  float x[KEEP][4], gw[KEEP][4];
  auto load = [&](int slot, float (&v)[4]) {
    load_numbers<float, 4, (PER > 0)>(xr + 4 * slot, H - 4 * slot, v);
    if (dr) {
      float d[4];
      load_numbers<TA, 4, (PER > 0)>(dr + 4 * slot, H - 4 * slot, d);
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const f32x2 sum = fma2(pair2(delta_scale, delta_scale), pair2(d[j], d[j + 1]), pair2(v[j], v[j + 1]));
        v[j] = low2(sum), v[j + 1] = high2(sum);
      }
    }
  };
  auto add_squares = [&](const float (&v)[4]) {
#pragma unroll
    for (int j = 0; j < 4; j += 2) ss = fma2(pair2(v[j], v[j + 1]), pair2(v[j], v[j + 1]), ss);
  };
  if constexpr (PER > 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int slot = threadIdx.x + i * blockDim.x;
      if (slot < slots) load(slot, x[i]);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {                         // the gains too in front of the first store, which they could not pass
      const int slot = threadIdx.x + i * blockDim.x;
      if (slot < slots) load_numbers<float, 4, true>(gain + 4 * slot, H - 4 * slot, gw[i]);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int slot = threadIdx.x + i * blockDim.x;
      if (slot >= slots) continue;
      if (so && 4 * slot < H) store_vec<float, 4>(so + 4 * slot, x[i]);
      add_squares(x[i]);
    }
  } else {
    for (int slot = threadIdx.x; slot < slots; slot += blockDim.x) {
      load(slot, x[0]);
      add_squares(x[0]);
    }
  }
  // (inside a warp additions of 32 bits, whose errors are independent from warp to warp and average out, across warps of 64)
  const double mean = block_sum64((double)warp_sum(low2(ss) + high2(ss)), red) * inv_h + (double)eps;
  const bool extreme = !((float)mean > kLeastMean && (float)mean < kMostMean);
  const float2 inv = inverse_root(mean);
  const RowFactor factor = {pair2(inv.x, inv.x), pair2(inv.y, inv.y), pair2(-inv.x, -inv.x), pair2(-inv.y, -inv.y)};
  if constexpr (PER > 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int slot = threadIdx.x + i * blockDim.x;        // whole warps: slots and threads are multiples of 32
      if (slot < slots) finish_four(x[i], gw[i], factor, codes, scales, (size_t)row * kb, slot);
    }
  } else {
    for (int slot = threadIdx.x; slot < slots; slot += blockDim.x) {
      load(slot, x[0]);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (so && 4 * slot + j < H) so[4 * slot + j] = x[0][j];
      load_numbers<float, 4, false>(gain + 4 * slot, H - 4 * slot, gw[0]);
      finish_four(x[0], gw[0], factor, codes, scales, (size_t)row * kb, slot);
    }
  }
  if (extreme) extreme_row<TA>(so ? so : xr, so ? nullptr : dr, delta_scale, gain, codes + (size_t)row * kb * kGroup, scales + (size_t)row * kb, H, kb, inv_h, eps, red);
}

// ------------------------------------------------------------------ gate
// y = act(gate) * up from float32 sums [rows, 256 nb] whose columns are 128 of the gate, 128 of the other, and so on: a warp has a group.
__global__ void __launch_bounds__(256) act_mul_q8_kernel(const float* sums, uint8_t* codes, uint8_t* scales, long groups, int act) {
  pdl_launch_dependents();
  pdl_wait();
  const long g = ((long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (g >= groups) return;
  float gate[4], v[4];
  load_vec<float, 4>(sums + g * 2 * kGroup + 4 * lane, gate);
  load_vec<float, 4>(sums + g * 2 * kGroup + kGroup + 4 * lane, v);
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] *= act == 0 ? q8_silu(gate[j]) : q8_gelu_tanh(gate[j]);
  uint32_t w[1];
  const float s = group_codes<32, 4>(v, w);
  *reinterpret_cast<uint32_t*>(codes + (size_t)g * kGroup + 4 * lane) = w[0];
  if (lane == 0) scales[g] = exponent_byte(s);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
int blocks_of(int n) { return (int)(((long)n + kGroup - 1) / kGroup); }

template <typename T>
int quantize_rows(const void* x, long row_stride, void* codes, void* scales, int M, int K, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T), per_block = 256 / (kGroup / V) * kAtOnce;
  const int kb = blocks_of(K);
  const long groups = (long)M * kb, blocks = (groups + per_block - 1) / per_block;
  if (groups + per_block > 0x7fffffffl) return ARLE_E_UNSUPPORTED;
  const bool fast = K % V == 0 && aligned16(x) && (M == 1 || row_stride % V == 0);
  // magic = (2^(31 + shift) + e) / kb with e < kb <= 2^shift, so for g below 2^31 g magic / 2^(31 + shift) is g / kb and less than 1 / kb more
  int shift = 0;
  while ((1l << shift) < kb) ++shift;
  const uint32_t magic = (uint32_t)(((1ull << (31 + shift)) + kb - 1) / kb);
  launch_early(fast ? quantize_rows_kernel<T, true> : quantize_rows_kernel<T, false>, dim3((unsigned)blocks), dim3(256), 0, s, 1, (const T*)x, row_stride,
                (uint8_t*)codes, (uint8_t*)scales, (uint32_t)groups, K, (uint32_t)kb, magic, shift);
  return launch_status();
}

template <typename T>
int quantize_weight(const void* w, long row_stride, void* codes, void* scales, int N, int K, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const int kb = blocks_of(K), nb = blocks_of(N);
  if (nb > 65535) return ARLE_E_UNSUPPORTED;
  const bool fast = K % V == 0 && aligned16(w) && (N == 1 || row_stride % V == 0);
  launch_early(fast ? quantize_weight_kernel<T, true> : quantize_weight_kernel<T, false>, dim3(kb, nb), dim3(256), 0, s, 1, (const T*)w, row_stride,
                (uint8_t*)codes, (float*)scales, N, K, kb);
  return launch_status();
}

template <typename TA>
int rmsnorm(const float* resid, const void* delta, const float* gain, float* sum_out, void* codes, void* scales, int M, int H, float eps, float delta_scale,
            cudaStream_t s) {
  const int kb = blocks_of(H);
  const bool vec = H % 4 == 0 && aligned16(resid) && aligned16(gain) && ((uintptr_t)delta % (4 * sizeof(TA))) == 0 && aligned16(sum_out);
  auto kern = rmsnorm_q8_kernel<TA, 0>;
  int threads = kb >= 32 ? 1024 : 32 * kb;
  if (vec && kb <= 128) {
    // few rows: as many threads as the row has pieces, the shortest way through it; many: two pieces a thread, so that three blocks of 5,120 numbers are on an SM
    // (four pieces, 48 registers and four blocks of half the threads: 58 us for 5,003 rows; one piece for 4,096 rows of 4,096: 42, two 35, four 39)
    const int per = M <= 256 || kb > 64 ? (kb + 31) / 32 : 2;
    threads = 32 * ((kb + per - 1) / per);
    kern = per == 1 ? rmsnorm_q8_kernel<TA, 1> : per == 2 ? rmsnorm_q8_kernel<TA, 2> : rmsnorm_q8_kernel<TA, 4>;
  }
  launch_early(kern, dim3(M), dim3(threads), 0, s, 1, resid, (const TA*)delta, gain, sum_out, (uint8_t*)codes, (uint8_t*)scales, H, kb, 1.0 / H, eps,
                delta_scale);
  return launch_status();
}

}  // namespace

// x [M, K] (dtype 0 float32, 1 bfloat16; rows row_stride apart) -> codes [M, 128 ceil(K / 128)] on a 16-byte boundary, scales [M, ceil(K / 128)].
ARLE_API int arle_quantize_q8(const void* x, int dtype, long row_stride, void* codes, void* scales, int M, int K, cudaStream_t s) {
  if (M <= 0) return 0;
  if (K <= 0 || !aligned16(codes)) return ARLE_E_BADARG;
  if (dtype == 0) return quantize_rows<float>(x, row_stride, codes, scales, M, K, s);
  if (dtype == 1) return quantize_rows<__nv_bfloat16>(x, row_stride, codes, scales, M, K, s);
  return ARLE_E_BADARG;
}

// w [N, K] -> codes [N, 128 ceil(K / 128)], float32 scales [ceil(N / 128), ceil(K / 128)].
ARLE_API int arle_quantize_weight_q8(const void* w, int dtype, long row_stride, void* codes, void* scales, int N, int K, cudaStream_t s) {
  if (N <= 0) return 0;
  if (K <= 0 || !aligned16(codes)) return ARLE_E_BADARG;
  if (dtype == 0) return quantize_weight<float>(w, row_stride, codes, scales, N, K, s);
  if (dtype == 1) return quantize_weight<__nv_bfloat16>(w, row_stride, codes, scales, N, K, s);
  return ARLE_E_BADARG;
}

// x = resid + delta_scale * delta (delta may be null); sum_out = x (null: not written; may be resid); codes and scales of x * rsqrt(mean(x^2) + eps) * gain.
ARLE_API int arle_rmsnorm_q8(const float* resid, const void* delta, int dtype, const float* gain, float* sum_out, void* codes, void* scales, int M, int H,
                             float eps, float delta_scale, cudaStream_t s) {
  if (M <= 0) return 0;
  if (H <= 0 || !aligned16(codes)) return ARLE_E_BADARG;
  if (dtype == 0) return rmsnorm<float>(resid, delta, gain, sum_out, codes, scales, M, H, eps, delta_scale, s);
  if (dtype == 1) return rmsnorm<__nv_bfloat16>(resid, delta, gain, sum_out, codes, scales, M, H, eps, delta_scale, s);
  return ARLE_E_BADARG;
}

// sums [M, 256 nb] float32 -> codes [M, 128 nb], scales [M, nb]; act 0 silu, 1 the tanh form of gelu.
ARLE_API int arle_act_mul_q8(const float* sums, void* codes, void* scales, int M, int nb, int act, cudaStream_t s) {
  if (M <= 0 || nb <= 0) return 0;
  if (act < 0 || act > 1 || !aligned16(sums) || !aligned16(codes)) return ARLE_E_BADARG;
  const long groups = (long)M * nb, blocks = (groups + 7) / 8;
  if (blocks > 0x7fffffffl) return ARLE_E_UNSUPPORTED;
  launch_early(act_mul_q8_kernel, dim3((unsigned)blocks), dim3(256), 0, s, 1, sums, (uint8_t*)codes, (uint8_t*)scales, groups, act);
  return launch_status();
}
