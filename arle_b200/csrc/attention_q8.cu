// Paged causal attention over the 8-bit cache (q8.cuh), the general form: any head size up to 256, values of their own width, any page size, any number
// of heads and groups, float32 or bfloat16 queries, float32 arithmetic throughout.
//     s_j = scale * k_scale[page of j] * (q . k_code_j);   out = sum_j exp(s_j - m) v_scale[page of j] v_code_j / (sum_j exp(s_j - m) + exp(sink - m))
// over the keys j that the query at position p sees (p - window < j <= p), m the largest score; a query that sees no key gets zeros.
// One block per (token, query head); warp w takes tiles w, w + 4, ... of 32 keys counted from the first visible one and the partial results are merged at
// the end, so a token's order of sums depends on its first key and position alone.  It serves what attention_q8_decode.cu and the prompt kernels do not
// take and is their yardstick; bound by its FFMA instructions.
#include "q8.cuh"
using namespace arle;

namespace {

constexpr int kWarps = 4;
constexpr int kMaxD = 8;      // widths up to 256

template <typename T>
__global__ void attention_q8_kernel(const T* __restrict__ q, int q_row_stride, T* __restrict__ out, const uint8_t* __restrict__ k_cache,
                                    const uint8_t* __restrict__ v_cache, const float* __restrict__ k_scale, const float* __restrict__ v_scale,
                                    const int* __restrict__ positions, const int* __restrict__ row_of_token, const int* __restrict__ block_table, int bt_stride,
                                    int nq, int nkv, int hd, int vd, int page_size, float scale, int window, const float* __restrict__ sinks) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ __align__(16) float qs[256];
  __shared__ float acc_s[kWarps][256];
  __shared__ float m_s[kWarps], l_s[kWarps];
  const int t = blockIdx.x, h = blockIdx.y, w = threadIdx.x >> 5, lane = threadIdx.x & 31, kvh = h / (nq / nkv);
  const int pos = positions[t], lo = pos >= 0 ? first_visible_key(pos, window, 0) : 0;
  const int* bt = block_table + (size_t)row_of_token[t] * bt_stride;
  const int nvis = pos - lo + 1;
  const T* qp = q + (size_t)t * q_row_stride + (size_t)h * hd;
  for (int e = threadIdx.x; e < hd; e += blockDim.x) qs[e] = to_f32(qp[e]) * scale;
  __syncthreads();

  float m = -INFINITY, l = 0.f, acc[kMaxD];
#pragma unroll
  for (int i = 0; i < kMaxD; ++i) acc[i] = 0.f;
  const bool quads = (hd & 3) == 0;
  for (int i0 = w * 32; i0 < nvis; i0 += kWarps * 32) {
    const int j = lo + i0 + lane;
    float sc = -INFINITY, vs = 0.f;
    long vrow = 0;
    if (i0 + lane < nvis) {
      const int page = bt[j / page_size];
      const long row = ((long)page * nkv + kvh) * page_size + j % page_size;
      const uint8_t* kp = k_cache + row * hd;
      float d = 0.f;
      if (quads) {
        for (int e = 0; e < hd; e += 4) {
          const uint32_t c = *reinterpret_cast<const uint32_t*>(kp + e);
          const float2 a = q8_float2(c & 0xffffu), b = q8_float2(c >> 16);
          d = fmaf(qs[e], a.x, d);
          d = fmaf(qs[e + 1], a.y, d);
          d = fmaf(qs[e + 2], b.x, d);
          d = fmaf(qs[e + 3], b.y, d);
        }
      } else {
        for (int e = 0; e < hd; ++e) d = fmaf(qs[e], q8_float(kp[e]), d);
      }
      sc = d * k_scale[(long)page * nkv + kvh];
      vs = v_scale[(long)page * nkv + kvh];
      vrow = row * vd;
    }
    const float m_new = fmaxf(m, warp_max(sc)), base = m_new == -INFINITY ? 0.f : m_new;      // scores that are all -infinity: weights of zero, not NaN
    const float p = i0 + lane < nvis ? expf(sc - base) : 0.f, corr = expf(m - base);
    l = l * corr + warp_sum(p);
#pragma unroll
    for (int i = 0; i < kMaxD; ++i) acc[i] *= corr;
    m = m_new;
    const float pv = p * vs;
    const int nvalid = min(32, nvis - i0);
    for (int jj = 0; jj < nvalid; ++jj) {
      const float pj = __shfl_sync(0xffffffffu, pv, jj);
      const uint8_t* vp = v_cache + __shfl_sync(0xffffffffu, vrow, jj);
#pragma unroll
      for (int i = 0; i < kMaxD; ++i) {
        const int d = lane + 32 * i;
        if (d < vd) acc[i] = fmaf(pj, q8_float(vp[d]), acc[i]);
      }
    }
  }
  if (lane == 0) {
    m_s[w] = m;
    l_s[w] = l;
  }
#pragma unroll
  for (int i = 0; i < kMaxD; ++i)
    if (lane + 32 * i < vd) acc_s[w][lane + 32 * i] = acc[i];
  __syncthreads();
  const float sink = sinks ? sinks[h] : -INFINITY;
  float mm = sink;
  for (int i = 0; i < kWarps; ++i) mm = fmaxf(mm, m_s[i]);
  const float base = mm == -INFINITY ? 0.f : mm;
  float f[kWarps], ll = expf(sink - base);
  for (int i = 0; i < kWarps; ++i) {
    f[i] = expf(m_s[i] - base);
    ll += l_s[i] * f[i];
  }
  T* op = out + ((size_t)t * nq + h) * vd;
  for (int d = threadIdx.x; d < vd; d += blockDim.x) {
    float o = 0.f;
    for (int i = 0; i < kWarps; ++i) o += acc_s[i][d] * f[i];
    op[d] = from_f32<T>(nvis > 0 ? o / ll : 0.f);
  }
}

}  // namespace

ARLE_API int arle_attention_q8(const void* q, int q_row_stride, void* out, int dtype, const void* k_cache, const void* v_cache, const float* k_scale,
                               const float* v_scale, const int* positions, const int* row_of_token, const int* block_table, int bt_stride, int nq, int nkv, int hd,
                               int vd, int page_size, float scale, int window, const float* sinks, int tokens, cudaStream_t s) {
  if (tokens <= 0) return 0;
  if (hd <= 0 || hd > 256 || vd <= 0 || vd > 256 || nkv <= 0 || nq <= 0 || nq % nkv || nq > 65535 || page_size <= 0) return ARLE_E_UNSUPPORTED;
  const dim3 grid(tokens, nq), block(kWarps * 32);
  if (dtype == 0)
    launch_kernel(attention_q8_kernel<float>, grid, block, 0, s, 1, (const float*)q, q_row_stride, (float*)out, (const uint8_t*)k_cache, (const uint8_t*)v_cache,
                  k_scale, v_scale, positions, row_of_token, block_table, bt_stride, nq, nkv, hd, vd, page_size, scale, window, sinks);
  else if (dtype == 1)
    launch_kernel(attention_q8_kernel<__nv_bfloat16>, grid, block, 0, s, 1, (const __nv_bfloat16*)q, q_row_stride, (__nv_bfloat16*)out,
                  (const uint8_t*)k_cache, (const uint8_t*)v_cache, k_scale, v_scale, positions, row_of_token, block_table, bt_stride, nq, nkv, hd, vd, page_size,
                  scale, window, sinks);
  else
    return ARLE_E_BADARG;
  return launch_status();
}
