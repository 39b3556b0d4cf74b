// Keys and values of a step's tokens into the 8-bit cache (q8.cuh), and pages of it back into bfloat16.
//
// store: token t goes to place slot_mapping[t] = page * page_size + offset; a negative place, or one behind the cache, stores nothing.  Consecutive
// tokens with consecutive places of one page are a run; a run starts at offset 0, where a page begins, or where a request's new tokens begin.  Per run
// and head, with a the largest finite |x| of its numbers and s(a) the scale that carries it:
//     s' = s(a) for a run from offset 0, else max(s, s(a));   codes in front of the run: rne(code * s / s');   new codes: rne(x / s')
// One group of `warps` warps owns a run of one head of the keys or the values, so the page's scale and older codes are read and written by one owner.
// A page of up to 2,048 numbers a warp stays in registers between the maximum and the rounding (one read of x); what is larger is read again (from L2).
// The kernel is bound by the latency of its three dependent reads (place, numbers, stores) for decoded tokens and by DRAM for prompts.
#include "q8.cuh"
using namespace arle;

namespace {

struct StoreSide {
  const void* x;
  int row_stride, width;
  uint8_t* cache;
  float* scale;
};

__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= 3.4028234663852886e38f ? a : 0.f;      // neither infinities nor NaN
}

template <typename T, int VEC>
__device__ __forceinline__ float most_of(const Pack<T, VEC>& p, float most) {
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

// A group has `warps` warps.  `chunk`: tokens among which a group looks for the starts of runs (at most 32).  VEC: numbers of a load, 16 bytes or one.
template <typename T, int VEC>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 2) store_q8_kernel(StoreSide ks, StoreSide vs, const int* __restrict__ slot_mapping, int tokens, int chunk, int nkv, int page_size,
                                                       long places, int warps, long groups) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kKept = VEC == 1 ? 1 : 64 / VEC;      // loads a lane keeps: 64 numbers
  __shared__ float most_s[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int lane_g = warps == 1 ? lane : threadIdx.x, size_g = warps * 32;
  const long group = warps == 1 ? (long)blockIdx.x * (blockDim.x >> 5) + warp : blockIdx.x;
  if (group >= groups) return;
  const StoreSide& side = (group & 1) ? vs : ks;
  const int head = (int)((group >> 1) % nkv), t0 = (int)((group >> 1) / nkv) * chunk;
  const int hd = side.width;
  const T* x = reinterpret_cast<const T*>(side.x) + (long)head * hd;

  // places of the chunk's tokens and of those behind it, one a lane
  const int s = t0 + lane < tokens ? slot_mapping[t0 + lane] : -1;
  int before = __shfl_up_sync(0xffffffffu, s, 1);
  if (lane == 0) before = t0 > 0 ? slot_mapping[t0 - 1] : -2;
  const bool held = s >= 0 && s < places;
  const bool first = held && (s % page_size == 0 || before != s - 1 || t0 + lane == 0);
  const unsigned goes_on = __ballot_sync(0xffffffffu, held && !first);
  unsigned starts = __ballot_sync(0xffffffffu, first && lane < chunk);
  const int per_row = hd / VEC;                       // loads of a row
  const bool even = size_g % per_row == 0;            // a lane keeps its column
  const int row0 = lane_g / per_row, col0 = lane_g - row0 * per_row, row_step = size_g / per_row;

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
    auto load = [&](int i) {
      const int e = i * size_g + lane_g;
      const int row = even ? row0 + i * row_step : e / per_row, col = even ? col0 : e - row * per_row;
      return *reinterpret_cast<const Pack<T, VEC>*>(rows + (long)row * side.row_stride + col * VEC);
    };
    auto to = [&](int i) { return codes + (long)off * hd + (long)(i * size_g + lane_g) * VEC; };

    Pack<T, VEC> kept[kKept];
    float most = 0.f;
    const bool once = loads <= kKept * size_g;
    if (once) {
#pragma unroll
      for (int i = 0; i < kKept; ++i)
        if (i * size_g + lane_g < loads) kept[i] = load(i);
#pragma unroll
      for (int i = 0; i < kKept; ++i)
        if (i * size_g + lane_g < loads) most = most_of(kept[i], most);
    } else {
#pragma unroll 4
      for (int i = 0; i * size_g + lane_g < loads; ++i) most = most_of(load(i), most);
    }
    most = warp_max(most);
    if (warps > 1) {
      __syncthreads();
      if (lane == 0) most_s[warp] = most;
      __syncthreads();
      for (int i = 0; i < warps; ++i) most = fmaxf(most, most_s[i]);
    }
    const float now = fmaxf(older, q8_scale(most)), inv = 1.0f / now;
    if (once) {
#pragma unroll
      for (int i = 0; i < kKept; ++i)
        if (i * size_g + lane_g < loads) put(to(i), kept[i], inv);
    } else {
#pragma unroll 4
      for (int i = 0; i * size_g + lane_g < loads; ++i) put(to(i), load(i), inv);
    }
    if (off && now == older) continue;
    if (off) {                                        // the page's older codes follow its scale
      const float by = older * inv;
      for (int e = lane_g; e < off * hd; e += size_g) {
        if constexpr (VEC == 1) {
          codes[e] = (uint8_t)q8_codes2(q8_float(codes[e]) * by, 0.f);
        } else {
          if (e * 4 >= off * hd) break;
          uint32_t* w = reinterpret_cast<uint32_t*>(codes) + e;
          const float2 a = q8_float2(*w & 0xffffu), b = q8_float2(*w >> 16);
          *w = q8_codes4(a.x * by, a.y * by, b.x * by, b.y * by);
        }
      }
    }
    if (lane_g == 0) *scale = now;
  }
}

template <typename T>
int launch_store(const StoreSide& k, const StoreSide& v, const int* slot_mapping, int tokens, int nkv, int page_size, long places, cudaStream_t s) {
  constexpr int VEC = 16 / sizeof(T);
  bool wide = true;
  for (const StoreSide* x : {&k, &v}) wide = wide && x->width % VEC == 0 && x->row_stride % VEC == 0 && (uintptr_t)x->x % 16 == 0 && (uintptr_t)x->cache % 8 == 0;
  const int chunk = tokens <= 512 ? 1 : 16;
  int warps = 1;
  while (warps < 8 && (long)warps * 2048 < (long)page_size * (k.width > v.width ? k.width : v.width)) warps *= 2;
  const long groups = (long)((tokens + chunk - 1) / chunk) * nkv * 2;
  const int threads = warps == 1 ? 128 : warps * 32;
  const long blocks = warps == 1 ? (groups + 3) / 4 : groups;
  if (blocks > 0x7fffffffL) return ARLE_E_UNSUPPORTED;
  launch_kernel(wide ? store_q8_kernel<T, VEC> : store_q8_kernel<T, 1>, dim3((unsigned)blocks), dim3(threads), 0, s, 1, k, v, slot_mapping, tokens, chunk, nkv,
                page_size, places, warps, groups);
  return launch_status();
}

// expand: the keys and values that rows with at least `least` queries see, as bfloat16 pages of 64 tokens [pages, nkv, 64, width] with a block table of
// their own, for the prompt kernels: a code is exact in bfloat16, and so is its product with a power of two.  Row r's pages follow those of the rows in
// front of it; its table names them at their logical places (page j holds tokens 64 j ...), -1 elsewhere.  Places behind the row's last token are zeros.
// A block per page and head, bound by DRAM (one byte in, two out).
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
    if (tid == 0) t[logical] = page;
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
  if (nkv <= 0 || hd <= 0 || vd <= 0 || page_size <= 0 || hd > 256 || vd > 256) return ARLE_E_UNSUPPORTED;
  if (pages * page_size > 0x7fffffffL) return ARLE_E_UNSUPPORTED;      // places are 32-bit
  const StoreSide ks{k, k_stride, hd, (uint8_t*)k_cache, k_scale}, vs{v, v_stride, vd, (uint8_t*)v_cache, v_scale};
  if (dtype == 0) return launch_store<float>(ks, vs, slot_mapping, tokens, nkv, page_size, pages * page_size, s);
  if (dtype == 1) return launch_store<__nv_bfloat16>(ks, vs, slot_mapping, tokens, nkv, page_size, pages * page_size, s);
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
