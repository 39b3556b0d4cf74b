// Keys and values of a step's tokens into the 8-bit cache (q8.cuh), and pages of it back into bfloat16.
//
// store: token t goes to place slot_mapping[t] = page * page_size + offset; a negative place, or one behind the cache, stores nothing.  Consecutive
// tokens with consecutive places of one page are a run; a run starts at offset 0, where a page begins, or where a request's new tokens begin.  Per run
// and head, with a the largest finite |x| of its numbers and s(a) the scale that carries it:
//     s' = s(a) for a run from offset 0, else max(s, s(a));   codes in front of the run: rne(code * s / s');   new codes: rne(x / s')
// One group of `warps` warps owns a run of one head of the keys or the values, so the page's scale and older codes are read and written by one owner.
// A page of up to 2,048 numbers a warp stays in registers between the maximum and the rounding (one read of x); what is larger is read again (from L2).
// Decoded tokens are bound by the latency of three dependent accesses (place, numbers, codes): 2.0 us for one token, 2.1 us for 64, where
// their pages' scales hold them; with all scales growing the rounding of older codes takes 15 us at the end of 64 pages of 16, 55 with pages of 64.  Prompts come near
// DRAM's rate: 15,000 tokens of 8 heads of 128 in 20.7 us, 4.7 TB/s; what is left is instructions (five for two numbers in the rounding alone).
#include "q8.cuh"
using namespace arle;

namespace {

struct StoreSide {
  const void* x;
  int row_stride, width;
  int per_row, row_step;      // loads of a row; rows between a lane's loads, 0 where it does not keep its column
  uint8_t* cache;
  float* scale;
};

__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= 3.4028234663852886e38f ? a : 0.f;      // neither infinities nor NaN
}

__device__ __forceinline__ float reciprocal(float s) {      // exactly, of a power of two
  const uint32_t b = __float_as_uint(s);
  return (b & 0x7fffffu) == 0 && b >= (1u << 23) && b < (254u << 23) ? __uint_as_float((254u << 23) - b) : 1.0f / s;
}

// The largest |x| of the loads taken in, of the finite ones.  Bits of numbers without their signs are in the order of the numbers, so the maximum is taken
// over whole words (two bfloat16 at a time); where it comes out as an infinity or a NaN the loads are gone through once more.
template <typename T, int VEC>
struct Most {
  uint32_t bits = 0;
  __device__ __forceinline__ void take(const Pack<T, VEC>& p) {
    if constexpr (VEC == 1) {
      bits = max(bits, __float_as_uint(finite_abs(to_f32(p.e[0]))));
    } else {
      const uint4 w = *reinterpret_cast<const uint4*>(&p);
      if constexpr (sizeof(T) == 2)
        bits = __vmaxu2(__vmaxu2(bits, __vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu)), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
      else
        bits = max(max(bits, max(w.x & 0x7fffffffu, w.y & 0x7fffffffu)), max(w.z & 0x7fffffffu, w.w & 0x7fffffffu));
    }
  }
  __device__ __forceinline__ float value() const {
    if constexpr (VEC > 1 && sizeof(T) == 2) return __uint_as_float(max(bits & 0xffffu, bits >> 16) << 16);
    else return __uint_as_float(bits);
  }
};
template <typename T, int VEC>
__device__ __forceinline__ float finite_of(const Pack<T, VEC>& p) {
  float most = 0.f;
#pragma unroll
  for (int j = 0; j < VEC; ++j) most = fmaxf(most, finite_abs(to_f32(p.e[j])));
  return most;
}

template <typename T, int VEC>
__device__ __forceinline__ void put(uint8_t* dst, const Pack<T, VEC>& p, float inv) {
  if constexpr (VEC == 1) {
    *dst = (uint8_t)q8_codes2(to_f32(p.e[0]) * inv, 0.f);
  } else {
    uint32_t w[VEC / 4];
#pragma unroll
    for (int j = 0; j < VEC / 4; ++j)
      w[j] = q8_codes4(to_f32(p.e[4 * j]) * inv, to_f32(p.e[4 * j + 1]) * inv, to_f32(p.e[4 * j + 2]) * inv, to_f32(p.e[4 * j + 3]) * inv);
    if constexpr (VEC == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(dst) = w[0];
  }
}

// A group has `warps` warps; where it has one, a block's warps take neighbouring heads (of the keys, then of the values).  `chunk`: tokens among which a
// group looks for the starts of runs (at most 31).  VEC: numbers of a load, 16 bytes or one.
template <typename T, int VEC>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 3 : 2) store_q8_kernel(StoreSide ks, StoreSide vs, const int* slot_mapping, int tokens, int chunk,
                                                                               int nkv, int page_size, int places, int warps) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kKept = VEC == 1 ? 1 : 64 / VEC;      // loads a lane keeps: 64 numbers
  __shared__ float most_s[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int lane_g = warps == 1 ? lane : threadIdx.x, size_g = warps * 32;
  const int unit = warps == 1 ? blockIdx.y * (blockDim.x >> 5) + warp : blockIdx.y;
  if (unit >= 2 * nkv) return;
  const StoreSide& side = unit < nkv ? ks : vs;
  const int head = unit < nkv ? unit : unit - nkv, t0 = blockIdx.x * chunk;
  const int hd = side.width;
  const T* x = reinterpret_cast<const T*>(side.x) + head * hd;

  // places of the chunk's tokens and of those behind it, one a lane
  const int s = t0 + lane < tokens ? slot_mapping[t0 + lane] : -1;
  int before = __shfl_up_sync(0xffffffffu, s, 1);
  if (lane == 0) before = t0 > 0 ? slot_mapping[t0 - 1] : -2;
  const bool held = s >= 0 && s < places;
  const bool first = held && (s % page_size == 0 || before != s - 1 || t0 + lane == 0);
  const unsigned goes_on = __ballot_sync(0xffffffffu, held && !first);
  unsigned starts = __ballot_sync(0xffffffffu, first && lane < chunk);
  const int per_row = side.per_row, row_step = side.row_step;

  auto rescale = [&](uint8_t* codes, int numbers, float by, int at, int step) {      // a page's older codes follow its scale
    if constexpr (VEC == 1) {
      for (int e = at; e < numbers; e += step) codes[e] = (uint8_t)q8_codes2(q8_float(codes[e]) * by, 0.f);
    } else {
      for (int e = at * 4; e < numbers; e += step * 4) {
        uint32_t* w = reinterpret_cast<uint32_t*>(codes + e);
        const float2 a = q8_float2(*w & 0xffffu), b = q8_float2(*w >> 16);
        *w = q8_codes4(a.x * by, a.y * by, b.x * by, b.y * by);
      }
    }
  };

  // runs of one token: eight lanes each
  const unsigned single = starts & ~(goes_on >> 1) & 0x7fffffffu;      // (what follows token 31 is not known here)
  starts &= ~single;
  for (int i0 = 0; single && i0 < chunk; i0 += size_g / 8) {
    const int i = i0 + lane_g / 8, sub = lane_g % 8;
    const bool mine = i < chunk && ((single >> i) & 1u);
    if (!__any_sync(0xffffffffu, mine)) continue;
    const int place = __shfl_sync(0xffffffffu, s, min(i, 31));
    const int page = mine ? place / page_size : 0, off = mine ? place - page * page_size : 0;
    const T* row = x + (long)(t0 + (mine ? i : 0)) * side.row_stride;
    uint8_t* codes = side.cache + ((long)page * nkv + head) * page_size * hd;
    float* scale = side.scale + (long)page * nkv + head;
    const float older = mine && off ? *scale : 0.f;
    constexpr int kRow = VEC == 1 ? 1 : 16 / VEC;       // loads of a lane that are kept: 128 numbers of a row
    Pack<T, VEC> kept[kRow];
    float most = 0.f;
    if (mine) {
      Most<T, VEC> all;
#pragma unroll
      for (int j = 0; j < kRow; ++j)
        if (j * 8 + sub < per_row) kept[j] = *reinterpret_cast<const Pack<T, VEC>*>(row + (j * 8 + sub) * VEC);
#pragma unroll
      for (int j = 0; j < kRow; ++j)
        if (j * 8 + sub < per_row) all.take(kept[j]);
      for (int e = kRow * 8 + sub; e < per_row; e += 8) all.take(*reinterpret_cast<const Pack<T, VEC>*>(row + e * VEC));
      most = all.value();
      if (!isfinite(most)) {
        most = 0.f;
        for (int e = sub; e < per_row; e += 8) most = fmaxf(most, finite_of(*reinterpret_cast<const Pack<T, VEC>*>(row + e * VEC)));
      }
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (!mine) continue;
    const float now = fmaxf(older, q8_scale(most)), inv = reciprocal(now);
    uint8_t* dst = codes + (long)off * hd;
#pragma unroll
    for (int j = 0; j < kRow; ++j)
      if (j * 8 + sub < per_row) put(dst + (j * 8 + sub) * VEC, kept[j], inv);
    for (int e = kRow * 8 + sub; e < per_row; e += 8) put(dst + e * VEC, *reinterpret_cast<const Pack<T, VEC>*>(row + e * VEC), inv);
    if (off && now == older) continue;
    if (off) rescale(codes, off * hd, older * inv, sub, 8);
    if (sub == 0) *scale = now;
  }

  while (starts) {
    const int at = __ffs(starts) - 1;
    starts &= starts - 1;
    const int place = __shfl_sync(0xffffffffu, s, at);
    const int page = place / page_size, off = place - page * page_size;
    // length of the run: the lanes behind its start that go on, and, where all do, further tokens, 32 at a time
    int n = __ffs(~(at == 31 ? 0u : goes_on >> (at + 1)));
    if (n == 32 - at)
      for (int more = 32; more == 32 && n < page_size - off; n += more) {
        const int t = t0 + at + n + lane;
        more = __ffs(~__ballot_sync(0xffffffffu, t < tokens && lane < page_size - off - n && slot_mapping[t] == place + n + lane)) - 1;
        if (more < 0) more = 32;
      }
    const T* rows = x + (long)(t0 + at) * side.row_stride;
    uint8_t* codes = side.cache + ((long)page * nkv + head) * page_size * hd;
    float* scale = side.scale + (long)page * nkv + head;
    const float older = off ? *scale : 0.f;
    const int loads = n * per_row;
    uint8_t* dst = codes + (long)off * hd + lane_g * VEC;
    Pack<T, VEC> kept[kKept];
    Most<T, VEC> all;
    auto at_load = [&](int e) { return *reinterpret_cast<const Pack<T, VEC>*>(rows + (long)(e / per_row) * side.row_stride + (e % per_row) * VEC); };
    const bool once = row_step && loads <= kKept * size_g, full = row_step && loads == kKept * size_g;      // a whole page of 2,048 numbers a warp: no conditions
    if (once) {
      const int row0 = lane_g / per_row, col0 = lane_g - row0 * per_row;
      const T* src = rows + (long)row0 * side.row_stride + col0 * VEC;
      const long step = (long)row_step * side.row_stride;
      if (full) {
#pragma unroll
        for (int i = 0; i < kKept; ++i) kept[i] = *reinterpret_cast<const Pack<T, VEC>*>(src + i * step);
#pragma unroll
        for (int i = 0; i < kKept; ++i) all.take(kept[i]);
      } else {
#pragma unroll
        for (int i = 0; i < kKept; ++i) {
          kept[i] = Pack<T, VEC>{};
          if (i * size_g + lane_g < loads) kept[i] = *reinterpret_cast<const Pack<T, VEC>*>(src + i * step);
        }
#pragma unroll
        for (int i = 0; i < kKept; ++i) all.take(kept[i]);
      }
    } else {
#pragma unroll 2
      for (int e = lane_g; e < loads; e += size_g) all.take(at_load(e));
    }
    float most = all.value();
    if (!isfinite(most)) {
      most = 0.f;
      for (int e = lane_g; e < loads; e += size_g) most = fmaxf(most, finite_of(at_load(e)));
    }
    most = warp_max(most);
    if (warps > 1) {
      __syncthreads();
      if (lane == 0) most_s[warp] = most;
      __syncthreads();
      for (int i = 0; i < warps; ++i) most = fmaxf(most, most_s[i]);
    }
    const float now = fmaxf(older, q8_scale(most)), inv = reciprocal(now);
    if (full) {
#pragma unroll
      for (int i = 0; i < kKept; ++i) put(dst + i * size_g * VEC, kept[i], inv);
    } else if (once) {
#pragma unroll
      for (int i = 0; i < kKept; ++i)
        if (i * size_g + lane_g < loads) put(dst + i * size_g * VEC, kept[i], inv);
    } else {
#pragma unroll 2
      for (int e = lane_g; e < loads; e += size_g) put(dst + (e - lane_g) * VEC, at_load(e), inv);
    }
    if (off && now == older) continue;
    if (off) rescale(codes, off * hd, older * inv, lane_g, size_g);
    if (lane_g == 0) *scale = now;
  }
}

template <typename T>
int launch_store(StoreSide k, StoreSide v, const int* slot_mapping, int tokens, int nkv, int page_size, int places, cudaStream_t s) {
  bool wide = true;
  for (const StoreSide* x : {&k, &v})
    wide = wide && x->width % (16 / sizeof(T)) == 0 && x->row_stride % (16 / sizeof(T)) == 0 && (uintptr_t)x->x % 16 == 0 && (uintptr_t)x->cache % 8 == 0;
  // Few tokens are likely to be decoded ones, a run each: four to a warp, eight lanes each.  Many are mostly prompts', whose runs are pages: with 16 to a warp
  // a page of 16 has a warp and none looks on (15,000 tokens: 20.7 us); 16 decoded ones among them are four passes of a warp.
  const int chunk = tokens <= 512 ? 4 : 16;
  int warps = 1;
  while (warps < 8 && (long)warps * 2048 < (long)page_size * (k.width > v.width ? k.width : v.width)) warps *= 2;
  for (StoreSide* x : {&k, &v}) {
    x->per_row = wide ? x->width / (int)(16 / sizeof(T)) : x->width;
    x->row_step = warps * 32 % x->per_row ? 0 : warps * 32 / x->per_row;
  }
  const int threads = warps == 1 ? 128 : warps * 32;
  const dim3 grid((tokens + chunk - 1) / chunk, warps == 1 ? (2 * nkv + 3) / 4 : 2 * nkv);
  // early: 15,000 tokens behind one another 22.6 -> 20.8 us, one token 7.4 -> 6.9 (launched one by one)
  launch_early(wide ? store_q8_kernel<T, 16 / sizeof(T)> : store_q8_kernel<T, 1>, grid, dim3(threads), 0, s, 1, k, v, slot_mapping, tokens, chunk, nkv, page_size,
                places, warps);
  return launch_status();
}

// expand: the keys and values that rows with at least `least` queries see, as bfloat16 pages of 64 tokens [pages, nkv, 64, width] with a block table of
// their own, for the prompt kernels: a code is exact in bfloat16, and so is its product with a power of two.  Row r's pages follow those of the rows in
// front of it; its table names them at their logical places (page j holds tokens 64 j ...), -1 elsewhere.  Places behind the row's last token are zeros.
// A block per page and head, bound by DRAM (one byte in, two out: 16,384 keys of 8 heads of 128 in 24 us, 4.2 TB/s) or by latency (2,100 keys: 5 us).
constexpr int kExpanded = 64;

struct ExpandArgs {
  const uint8_t *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  const int *q_indptr, *kv_lens, *block_table;
  int bt_stride, page_size, nkv, hd, window, rows, least;
  __nv_bfloat16 *k_out, *v_out;
  int* table_out;
  int table_width;
};

__device__ __forceinline__ int2 expanded_pages(const ExpandArgs& a, int r) {      // first logical page and the one behind the last
  const int n = a.q_indptr[r + 1] - a.q_indptr[r], kv = a.kv_lens[r];
  if (n < a.least || kv <= 0) return make_int2(0, 0);
  return make_int2(first_visible_key(max(kv - n, 0), a.window, 0) / kExpanded, (kv + kExpanded - 1) / kExpanded);
}

__global__ void __launch_bounds__(256) expand_q8_kernel(ExpandArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ int sum_s[8], row_s, at_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, head = blockIdx.y, page = blockIdx.x;
  const int each = (a.rows + 255) / 256, r0 = min(tid * each, a.rows), r1 = min(r0 + each, a.rows);
  if (tid == 0) row_s = -1;
  int mine = 0;
  for (int r = r0; r < r1; ++r) {
    const int2 p = expanded_pages(a, r);
    mine += p.y - p.x;
  }
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  if (lane == 31) sum_s[warp] = upto;
  __syncthreads();
  int front = upto - mine;
  for (int w = 0; w < warp; ++w) front += sum_s[w];
  if (page >= front && page < front + mine)
    for (int r = r0;; ++r) {
      const int2 p = expanded_pages(a, r);
      if (page < front + p.y - p.x) {
        row_s = r;
        at_s = front;
        break;
      }
      front += p.y - p.x;
    }
  __syncthreads();
  const int r = row_s;
  if (r < 0) return;
  const int2 span = expanded_pages(a, r);
  const int logical = span.x + page - at_s, kv = a.kv_lens[r], first = logical * kExpanded;
  if (head == 0) {
    int* t = a.table_out + (long)r * a.table_width;
    if (tid == 0 && logical < a.table_width) t[logical] = page;
    if (logical == span.x)
      for (int j = tid; j < a.table_width; j += 256)
        if (j < span.x || j >= span.y) t[j] = -1;
  }
  const int* bt = a.block_table + (long)r * a.bt_stride;
  const int parts = a.hd / 16;      // sixteen codes each
  const long to = ((long)page * a.nkv + head) * kExpanded * a.hd;
  for (int e = tid; e < kExpanded * parts; e += 256) {
    const int key = first + e / parts, part = e % parts;
    uint4 k = make_uint4(0, 0, 0, 0), v = k;
    float ks = 0.f, vs = 0.f;
    if (key < kv) {
      const int pg = bt[key / a.page_size];
      if (pg >= 0) {
        const long unit = (long)pg * a.nkv + head, from = (unit * a.page_size + key % a.page_size) * a.hd + part * 16;
        k = *reinterpret_cast<const uint4*>(a.k_cache + from);
        v = *reinterpret_cast<const uint4*>(a.v_cache + from);
        ks = a.k_scale[unit];
        vs = a.v_scale[unit];
      }
    }
    auto wide = [](const uint4& w, float by, __nv_bfloat16* dst) {
      const uint32_t x[4] = {w.x, w.y, w.z, w.w};
      uint32_t y[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 lo = q8_float2(x[i] & 0xffffu), hi = q8_float2(x[i] >> 16);
        const __nv_bfloat162 p = __floats2bfloat162_rn(lo.x * by, lo.y * by), q = __floats2bfloat162_rn(hi.x * by, hi.y * by);
        y[2 * i] = *reinterpret_cast<const uint32_t*>(&p);
        y[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&q);
      }
      reinterpret_cast<uint4*>(dst)[0] = make_uint4(y[0], y[1], y[2], y[3]);
      reinterpret_cast<uint4*>(dst)[1] = make_uint4(y[4], y[5], y[6], y[7]);
    };
    wide(k, ks, a.k_out + to + (long)(e / parts) * a.hd + part * 16);
    wide(v, vs, a.v_out + to + (long)(e / parts) * a.hd + part * 16);
  }
}

}  // namespace

// k [tokens, nkv * hd] and v [tokens, nkv * vd] (dtype, row strides in elements) into codes [pages, nkv, page_size, hd | vd] and scales [pages, nkv].
ARLE_API int arle_store_q8(const void* k, int k_stride, const void* v, int v_stride, int dtype, const int* slot_mapping, int tokens, void* k_cache, void* v_cache,
                           float* k_scale, float* v_scale, long pages, int nkv, int hd, int vd, int page_size, cudaStream_t s) {
  if (tokens <= 0) return 0;
  if (nkv <= 0 || hd <= 0 || vd <= 0 || page_size <= 0 || hd > 256 || vd > 256 || nkv > 16384) return ARLE_E_UNSUPPORTED;
  if (pages * page_size > 0x7fffffffL) return ARLE_E_UNSUPPORTED;      // places are 32-bit
  const StoreSide ks{k, k_stride, hd, 0, 0, (uint8_t*)k_cache, k_scale}, vs{v, v_stride, vd, 0, 0, (uint8_t*)v_cache, v_scale};
  if (dtype == 0) return launch_store<float>(ks, vs, slot_mapping, tokens, nkv, page_size, (int)(pages * page_size), s);
  if (dtype == 1) return launch_store<__nv_bfloat16>(ks, vs, slot_mapping, tokens, nkv, page_size, (int)(pages * page_size), s);
  return ARLE_E_BADARG;
}

// pages: the sum over the rows of the pages of 64 that they see (fewer blocks run than asked for if it is less).  Outputs as above; table_out
// [rows, table_width]; hd a multiple of 16.
ARLE_API int arle_expand_q8(const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale, const int* q_indptr, const int* kv_lens,
                            const int* block_table, int bt_stride, int page_size, int nkv, int hd, int window, int rows, int least, void* k_out, void* v_out,
                            int pages, int* table_out, int table_width, cudaStream_t s) {
  if (rows <= 0 || pages <= 0) return 0;
  if (hd <= 0 || hd % 16 || nkv <= 0 || nkv > 65535 || page_size <= 0 || table_width <= 0) return ARLE_E_UNSUPPORTED;
  const ExpandArgs a{(const uint8_t*)k_cache, (const uint8_t*)v_cache, k_scale, v_scale, q_indptr, kv_lens, block_table, bt_stride, page_size, nkv, hd, window,
                     rows, least, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, table_out, table_width};
  launch_kernel(expand_q8_kernel, dim3(pages, nkv), dim3(256), 0, s, 1, a);
  return launch_status();
}
