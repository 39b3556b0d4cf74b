// Paged causal attention over the 8-bit cache (q8.cuh), the general form: any head size up to 256, values of their own width, any page size, any number
// of heads and groups, float32 or bfloat16 queries, float32 arithmetic throughout.
//     s_j = scale * k_scale[page of j] * (q . k_code_j);   out = sum_j exp(s_j - m) v_scale[page of j] v_code_j / (sum_j exp(s_j - m) + exp(sink - m))
// over the keys j that the query at position p sees (p - window < j <= p), m the largest score; a query that sees no key gets zeros.  A page that is not
// there (-1) counts as keys and values of zeros, as in the other kernels: nothing is read for it, and an empty step's queries get zeros.
// One block per (token, query head); warp w takes tiles w, w + 8, ... of 32 keys counted from the first visible one and the partial results are merged at
// the end, so a token's order of sums depends on its first key and position alone.  In a tile a lane first has a key (whole rows of codes, 16 bytes a load),
// then four numbers of every value (one load a key, eight keys under way).  Two rows of 817
// keys with 8 heads of 128 take 15 us, 8 rows of 8,000 with 16 heads 152 us (byte loads, a key at a time: 108 and 1,456).
// It serves what attention_q8_decode.cu and the prompt kernels do not take and is their yardstick; bound by the latency of its loads where there are few
// tokens, by its conversions and FFMA instructions where there are many.
#include <type_traits>

#include "q8.cuh"
using namespace arle;

namespace {

constexpr int kWarps = 8;
constexpr int kQuads = 2;      // four numbers of a value each: widths up to 256
// The values' sums are taken in units of 2^24: values end at 2^128 (448 * 2^119), and what up to 2^24 keys add before the largest score is met, or before the
// division, stays in float32's range.  Exact, but for products below 2^-102.
constexpr float kUnit = 16777216.f;

// WIDE: keys of a multiple of 16 numbers, values of a multiple of 4, caches on 16-byte boundaries.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kWarps * 32) attention_q8_kernel(const T* __restrict__ q, int q_row_stride, T* __restrict__ out,
                                                                   const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache,
                                                                   const float* __restrict__ k_scale, const float* __restrict__ v_scale,
                                                                   const int* __restrict__ positions, const int* __restrict__ row_of_token,
                                                                   const int* __restrict__ block_table, int bt_stride, int nq, int nkv, int hd, int vd,
                                                                   int page_size, float scale, int window, const float* __restrict__ sinks) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ __align__(16) float qs[256];
  __shared__ __align__(16) float acc_s[kWarps][256];
  __shared__ float m_s[kWarps], l_s[kWarps], p_s[kWarps][32];
  __shared__ long row_s[kWarps][32];
  const int t = blockIdx.x, h = blockIdx.y, w = threadIdx.x >> 5, lane = threadIdx.x & 31, kvh = h / (nq / nkv);
  const int pos = positions[t], lo = pos >= 0 ? first_visible_key(pos, window, 0) : 0;
  const int* bt = block_table + (size_t)row_of_token[t] * bt_stride;
  const int nvis = pos - lo + 1;
  const T* qp = q + (size_t)t * q_row_stride + (size_t)h * hd;
  for (int e = threadIdx.x; e < hd; e += blockDim.x) qs[e] = to_f32(qp[e]) * scale;
  __syncthreads();

  float m = -INFINITY, l = 0.f, acc[kQuads][4];
#pragma unroll
  for (int i = 0; i < kQuads; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
  for (int i0 = w * 32; i0 < nvis; i0 += kWarps * 32) {
    const int j = lo + i0 + lane;
    const bool seen = i0 + lane < nvis;
    const int page = seen ? bt[j / page_size] : -1;
    float sc = seen ? 0.f : -INFINITY, vs = 0.f;
    long row = -1;
    if (page >= 0) {
      const long unit = (long)page * nkv + kvh;
      row = unit * page_size + j % page_size;
      const float ks = k_scale[unit];
      vs = v_scale[unit] * (1.f / kUnit);
      const uint8_t* kp = k_cache + row * hd;
      float d = 0.f;
      if constexpr (WIDE) {
#pragma unroll 4
        for (int e = 0; e < hd; e += 16) {
          const uint4 c4 = *reinterpret_cast<const uint4*>(kp + e);
          const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float4 qv = *reinterpret_cast<const float4*>(qs + e + 4 * x);
            const float2 a = q8_float2(c[x] & 0xffffu), b = q8_float2(c[x] >> 16);
            d = fmaf(qv.x, a.x, d);
            d = fmaf(qv.y, a.y, d);
            d = fmaf(qv.z, b.x, d);
            d = fmaf(qv.w, b.y, d);
          }
        }
      } else {
        for (int e = 0; e < hd; ++e) d = fmaf(qs[e], q8_float(kp[e]), d);
      }
      sc = d * ks;
    }
    const float m_new = fmaxf(m, warp_max(sc)), base = m_new == -INFINITY ? 0.f : m_new;      // scores that are all -infinity: weights of zero, not NaN
    const float p = seen ? expf(sc - base) : 0.f, corr = expf(m - base);
    l = l * corr + warp_sum(p);
#pragma unroll
    for (int i = 0; i < kQuads; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x) acc[i][x] *= corr;
    m = m_new;
    __syncwarp();
    p_s[w][lane] = page >= 0 ? p * vs : 0.f;
    row_s[w][lane] = row * vd;                       // negative: none
    __syncwarp();
    const int nvalid = min(32, nvis - i0);
    // all pages are there, mostly: asking key by key costs a third of the time (8 rows of 8,000 keys: 195 us instead of 152)
    auto add_values = [&](auto asked) {
      if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
          const int d = 4 * (lane + 32 * i);
          if (d < vd) {
            for (int j0 = 0; j0 < nvalid; j0 += 8) {
              uint32_t c[8];
#pragma unroll
              for (int x = 0; x < 8; ++x)
                c[x] = j0 + x < nvalid && (!asked.value || row_s[w][j0 + x] >= 0) ? *reinterpret_cast<const uint32_t*>(v_cache + row_s[w][j0 + x] + d) : 0u;
#pragma unroll
              for (int x = 0; x < 8; ++x) {
                const float pj = p_s[w][min(j0 + x, 31)];
                const float2 a = q8_float2(c[x] & 0xffffu), b = q8_float2(c[x] >> 16);
                acc[i][0] = fmaf(pj, a.x, acc[i][0]);
                acc[i][1] = fmaf(pj, a.y, acc[i][1]);
                acc[i][2] = fmaf(pj, b.x, acc[i][2]);
                acc[i][3] = fmaf(pj, b.y, acc[i][3]);
              }
            }
          }
        }
      } else {
        for (int jj = 0; jj < nvalid; ++jj) {
          if (asked.value && row_s[w][jj] < 0) continue;
          const float pj = p_s[w][jj];
          const uint8_t* vp = v_cache + row_s[w][jj];
#pragma unroll
          for (int i = 0; i < kQuads; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int d = 4 * (lane + 32 * i) + x;
              if (d < vd) acc[i][x] = fmaf(pj, q8_float(vp[d]), acc[i][x]);
            }
        }
      }
    };
    if (__all_sync(0xffffffffu, page >= 0 || !seen)) add_values(std::false_type{});
    else add_values(std::true_type{});
  }
  if (lane == 0) {
    m_s[w] = m;
    l_s[w] = l;
  }
#pragma unroll
  for (int i = 0; i < kQuads; ++i) *reinterpret_cast<float4*>(&acc_s[w][4 * (lane + 32 * i)]) = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
  __syncthreads();
  const float sink = sinks ? sinks[h] : -INFINITY;
  float mm = sink;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) mm = fmaxf(mm, m_s[i]);
  const float base = mm == -INFINITY ? 0.f : mm;
  float f[kWarps], ll = expf(sink - base);
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    f[i] = expf(m_s[i] - base);
    ll += l_s[i] * f[i];
  }
  T* op = out + ((size_t)t * nq + h) * vd;
  for (int d = threadIdx.x; d < vd; d += blockDim.x) {
    float o = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) o += acc_s[i][d] * f[i];
    op[d] = from_f32<T>(nvis > 0 ? o / ll * kUnit : 0.f);
  }
}

template <typename T>
void launch(const void* q, int q_row_stride, void* out, const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale, const int* positions,
            const int* row_of_token, const int* block_table, int bt_stride, int nq, int nkv, int hd, int vd, int page_size, float scale, int window, const float* sinks,
            int tokens, cudaStream_t s) {
  const bool wide = hd % 16 == 0 && vd % 4 == 0 && ((uintptr_t)k_cache | (uintptr_t)v_cache) % 16 == 0;
  launch_kernel(wide ? attention_q8_kernel<T, true> : attention_q8_kernel<T, false>, dim3(tokens, nq), dim3(kWarps * 32), 0, s, 1, (const T*)q, q_row_stride, (T*)out,
                (const uint8_t*)k_cache, (const uint8_t*)v_cache, k_scale, v_scale, positions, row_of_token, block_table, bt_stride, nq, nkv, hd, vd, page_size, scale,
                window, sinks);
}

}  // namespace

ARLE_API int arle_attention_q8(const void* q, int q_row_stride, void* out, int dtype, const void* k_cache, const void* v_cache, const float* k_scale,
                               const float* v_scale, const int* positions, const int* row_of_token, const int* block_table, int bt_stride, int nq, int nkv, int hd,
                               int vd, int page_size, float scale, int window, const float* sinks, int tokens, cudaStream_t s) {
  if (tokens <= 0) return 0;
  if (hd <= 0 || hd > 256 || vd <= 0 || vd > 256 || nkv <= 0 || nq <= 0 || nq % nkv || nq > 65535 || page_size <= 0) return ARLE_E_UNSUPPORTED;
  if (dtype == 0)
    launch<float>(q, q_row_stride, out, k_cache, v_cache, k_scale, v_scale, positions, row_of_token, block_table, bt_stride, nq, nkv, hd, vd, page_size, scale, window,
                  sinks, tokens, s);
  else if (dtype == 1)
    launch<__nv_bfloat16>(q, q_row_stride, out, k_cache, v_cache, k_scale, v_scale, positions, row_of_token, block_table, bt_stride, nq, nkv, hd, vd, page_size, scale,
                          window, sinks, tokens, s);
  else
    return ARLE_E_BADARG;
  return launch_status();
}
