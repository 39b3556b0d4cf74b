// Attention of decoded tokens (rows with one query) over the 8-bit cache (q8.cuh): bfloat16 queries, heads of 64 and 128, up to 16 query heads to a kv head.
//     s_j = scale * k_scale * (q . k_code_j);   out = sum_j exp(s_j) v_scale v_code_j / (sum_j exp(s_j) + exp(sink)),   kv_len - window <= j < kv_len
// A token reads every visible code once, so the kernel is built to stream codes at the rate of DRAM: 64 rows of up to 4,096 keys with 8 kv heads of 128 (374
// MB) take 66 us, 8 rows of up to 131,072 (1.3 GB) 207 us, 6.2 TB/s.  Some 12 us are latency whatever the keys: reading the rows' lengths, page ids and
// first tiles 3 to 6 us, joining sums 3; one row of 1,000 keys takes 8 us.
//
// Work: all rows' and heads' keys in blocks of 64 (128) are one line that a resident grid shares out evenly, whatever the rows' lengths; a CTA's piece of a
// (row, kv head) is summed on its own, and where a pair was cut the CTA that finishes its last piece joins the pieces in the order of keys (a counter per
// pair, which it leaves at zero).  Inside a piece warp w of four takes tiles w, w + 4, ... of 16 keys (32 of heads of 64); each warp has a ring of its own that
// cp.async fills, so nothing in the loop waits for another warp.
//
// Arithmetic: codes are exact in float16 (cvt), so both products run as mma.sync with float16 operands and float32 sums, keys as rows: S^T = K Q^T and
// O^T = V^T P^T, eight queries to an instruction (padding of G query heads to 8 and not to 16).  q is exact in float16 once a power of two has brought
// its largest number to [2^14, 2^15); numbers 2^-38 times that are lost.  Scores, sums and the maximum that the exponentials are taken against are float32.
// That maximum is followed only where a score passes it by more than kSlack (in log2): the weights stay below 2^kSlack, most tiles need no reduction across
// lanes and no correction of the sums.  A weight times its key's v_scale is rounded to float16, 11 bits (bfloat16 would keep 8), relative to a second
// maximum, of weight times scale, that is followed in the same way: at most 2^(kSlack + kUp) = 2^15, in whole down to 2^(-14 - kUp) of the largest.  So
// keys that carry a query's result keep their bits however much larger the values of other pages are.  The product is one exponential of the score plus
// the scale's logarithm: scales reach from 2^-100 (a page of zeros) to 2^119, and a weight that is zero in float32 times a factor that passes its range would
// be NaN.  The values' sums stay relative to the second maximum up to the last rounding, for the same reason.
// The order of the elements of a head among the k indices of S^T, and among the rows of O^T, is free as long as both operands agree: lane (g, c) owns
// numbers c * HD / 4 ... of a key and g * HD / 8 ... of the values, so a lane's codes are whole 16-byte reads (8 bytes for the values of heads of 64).
// Rows lie in shared memory with their 16-byte parts in an order turned by the key, which keeps those reads free of bank conflicts.
#include "mma_utils.cuh"
#include "q8.cuh"
using namespace arle;

namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kTile = 16;                 // keys of a product
// Products that a warp has in hand at a time (its tile): two where heads are small, so that a tile has as many bytes and its bookkeeping as much to do.
template <int HD> constexpr int kSub = HD == 64 ? 2 : 1;
template <int HD> constexpr int kKeys = kTile * kSub<HD>;           // keys of a warp's tile
template <int HD> constexpr int kBlock = kWarps * kKeys<HD>;        // keys of a block of work: 16 KB of codes
constexpr int kUp = 9;
constexpr float kSlack = 6.0f;
constexpr float kNone = -3.4028234663852886e38f;      // a maximum of nothing: finite, so that no difference of two is NaN

struct DecodeArgs {
  const __nv_bfloat16* q;
  int q_row_stride;
  __nv_bfloat16* out;
  const uint8_t *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  const int *q_indptr, *kv_lens, *block_table;
  int bt_stride;
  float *part_o, *part_ml;
  int* counters;
  int nq, nkv, page_size, ps_shift, window, rows;
  float scale_log2;
  const float* sinks;
  int beside;
  const int *positions, *row_of_token;      // null: rows are the step's rows; else its tokens, each by itself
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turned(uint32_t v) {      // an 8 x 8 matrix of 16-bit numbers, transposed across the warp
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {      // what is below 2^-126 is zero
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float log2_fast(float x) {      // of zero minus infinity
  float r;
  asm("lg2.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A row: its token, its keys, the block (on the grid of absolute positions) that its first visible key lies in, and how many blocks its query
// sees: none if the row has not exactly one query, one (which writes its zeros) if it has no keys.  By tokens a token is a row of the keys up to its own.
struct Row {
  int t, kv, first, nb, table;
};
template <int HD>
__device__ __forceinline__ Row row_of(const DecodeArgs& a, int r) {
  if (a.positions) {
    const int kv = a.positions[r] + 1, first = kv > 0 ? first_visible_key(kv - 1, a.window, 0) / kBlock<HD> : 0;
    return Row{r, kv, first, kv <= 0 ? 1 : (kv + kBlock<HD> - 1) / kBlock<HD> - first, a.row_of_token[r]};
  }
  const int t0 = a.q_indptr[r], t1 = a.q_indptr[r + 1], kv = a.kv_lens[r];
  const int first = kv > 0 ? first_visible_key(kv - 1, a.window, 0) / kBlock<HD> : 0;
  return Row{t0, kv, first, t1 - t0 != 1 ? 0 : kv <= 0 ? 1 : (kv + kBlock<HD> - 1) / kBlock<HD> - first, r};
}

constexpr int kPause = 6;      // blocks; see where the line is cut

template <int HD, int NT> struct Shape {
  static constexpr int kResident = NT == 1 ? 4 : 3;      // CTAs of an SM: 128 and 168 registers a thread
  static constexpr int kStages = NT == 1 ? 3 : 4;
  static constexpr int kStageBytes = 2 * kKeys<HD> * HD;
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kScales = kWarps * kStages * kSub<HD> * 32 * 4;
  static constexpr int kSmem = kRing + kScales;
  static constexpr int kPitch = HD + 8;      // of the partial results
};

// NT: query heads of a kv head in eights.  P16: pages of a multiple of 16 tokens, so that a tile lies in one page.
template <int HD, int NT, bool P16>
__device__ __forceinline__ void q8_decode(const DecodeArgs& a) {
  using S = Shape<HD, NT>;
  constexpr int SUB = kSub<HD>, NS = S::kStages, CH = HD / 16;      // 16-byte parts of a row
  constexpr int KS = HD / 16, MT = HD / 16;         // steps of 16 numbers of a head in S^T, tiles of 16 numbers in O^T
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int4 sum_s[kWarps];
  __shared__ int start_s[2], cut_s[2], last_s;
  __shared__ Row start_row;
  __shared__ float ml_s[kWarps][NT * 8][3];         // largest score, sum of weights, second maximum
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int G = a.nq / a.nkv, nkv = a.nkv;
  unsigned char* ring = smem + warp * NS * S::kStageBytes;
  float* scales = reinterpret_cast<float*>(smem + S::kRing) + warp * NS * SUB * 32;
  const uint32_t ring_u32 = smem_u32(ring), scales_u32 = smem_u32(scales);
  // where the lane's 16-byte parts of a tile go, beside i * 512: part i * 32 + lane is part lane % CH of key (i * 32 + lane) / CH
  uint32_t turned_at[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int key = (i * 32 + lane) / CH, turn = HD == 128 ? (key & 7) : ((key >> 1) & 3);
    turned_at[i] = key * HD + (((lane % CH) ^ turn) * 16) - i * 512;
  }

  // this CTA's share of the line, and the row where it begins
  const int each = (a.rows + kThreads - 1) / kThreads, r0 = min(tid * each, a.rows), r1 = min(r0 + each, a.rows);
  int mine = 0, mine_rows = 0, longest = 0;
  Row own{};                                       // the thread's first row
  for (int r = r1 - 1; r >= r0; --r) {
    own = row_of<HD>(a, r);
    mine += own.nb;
    mine_rows += own.nb > 0;
    longest = max(longest, own.nb);
  }
  int upto = mine, upto_rows = mine_rows;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, upto, o), y = __shfl_up_sync(0xffffffffu, upto_rows, o);
    if (lane >= o) upto += x, upto_rows += y;
  }
  longest = __reduce_max_sync(0xffffffffu, longest);
  if (lane == 31) sum_s[warp] = make_int4(upto, upto_rows, longest, 0);
  __syncthreads();
  int total = 0, total_rows = 0, front = upto - mine, front_rows = upto_rows - mine_rows;
  for (int w = 0; w < kWarps; ++w) {
    const int4 x = sum_s[w];
    if (w < warp) front += x.x, front_rows += x.y;
    total += x.x, total_rows += x.y;
    longest = max(longest, x.z);
  }
  // A CTA that goes on to another pair waits for that one's first tiles behind everybody's loads, about as long as `pause` blocks take it (6 us; 64 rows of
  // ragged lengths, CTAs of one, two and three pieces with the same keys: done after 51, 58 and 63 us).  So where shares are long a pair counts that
  // much more on the line, at its start; short shares are one piece each, mostly.
  const int pause = (total * nkv + (int)gridDim.x - 1) / (int)gridDim.x >= 4 * kPause ? kPause : 0;
  total = (total + pause * total_rows) * nkv;
  front = (front + pause * front_rows) * nkv;
  mine = (mine + pause * mine_rows) * nkv;
  // Cuts of the line: every `share` blocks, moved to the end, or else to the start, of the pair that they fall into where that is at most `slack` blocks
  // away: a piece costs its first tiles' latency and the joining beside its keys, and pairs shorter than a share stay whole.
  // The longest pair is in no more pieces than pay: a block takes a CTA alone some 0.5 us, and the CTA that joins reads G * HD numbers of every piece, one
  // after the other; share * 0.5 us + longest / share * G * 25 ns is least at 0.22 sqrt(longest * G).  (One row of 4,096 with 64 heads on 8: 21.3 us with
  // pieces of one block, 14.4 with four.)
  const int share = max((total + (int)gridDim.x - 1) / (int)gridDim.x, (int)(0.22f * sqrtf((float)longest * G) + 0.5f)), slack = min(3, (share + 1) / 2);
  if ((int)blockIdx.x * share >= total) return;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int at = ((int)blockIdx.x + i) * share;
    if (at >= total) {
      if (tid == 0) cut_s[i] = total;
    } else if (at >= front && at < front + mine) {
      int r = r0, row_at = front;
      Row x = own;
      for (;;) {
        const int n = x.nb > 0 ? (x.nb + pause) * nkv : 0;
        if (at < row_at + n) break;
        row_at += n;
        x = row_of<HD>(a, ++r);
      }
      const int from = (at - row_at) % (x.nb + pause), blk = max(0, from - pause), left = x.nb - blk;
      cut_s[i] = from == 0 ? at : left <= slack ? at - from + x.nb + pause : blk <= slack ? at - from : at;
      if (i == 0) {
        start_s[0] = r;
        start_s[1] = row_at;
        start_row = x;
      }
    }
  }
  __syncthreads();
  const int begin = cut_s[0], end = cut_s[1];
  if (begin >= end) return;
  int row = start_s[0], row_at = start_s[1];      // the row and where its blocks begin on the line
  Row at_row = start_row;

  // Sums lie in the order in which lanes have them, which keeps their way through shared memory free of bank conflicts: place p = 16 j + 2 g + b is
  // number g * HD / 8 + 2 j + b.  Four places' results (p a multiple of 4) of a head: sums of weights relative to 2^M, of values relative to 2^(MW - kUp);
  // none: the row has no keys.
  auto finish = [&](int t, int head, int p, float M, float L, float MW, const float4& O, bool none) {
    if (a.sinks) {
      const float sink = a.sinks[head] * 1.4426950408889634f, top = fmaxf(M, sink), base = fabsf(top) == INFINITY ? 0.f : top;
      L = L * exp2f(M - base) + exp2f(sink - base);
      M = top;
    }
    const float inv = none ? 0.f : exp2f(MW - (fabsf(M) == INFINITY ? 0.f : M) - kUp) / L;
    __nv_bfloat16* to = a.out + ((size_t)t * a.nq + head) * HD + (p % 16 / 2) * (HD / 8) + p / 16 * 2;
    *reinterpret_cast<__nv_bfloat162*>(to) = __floats2bfloat162_rn(O.x * inv, O.y * inv);
    *reinterpret_cast<__nv_bfloat162*>(to + HD / 8) = __floats2bfloat162_rn(O.z * inv, O.w * inv);
  };

  for (int pos = begin; pos < end;) {
    for (;;) {
      const int n = at_row.nb > 0 ? (at_row.nb + pause) * nkv : 0;
      if (pos < row_at + n) break;
      row_at += n;
      at_row = row_of<HD>(a, ++row);
    }
    const int nb = at_row.nb, t = at_row.t, kv = at_row.kv;
    const int h = (pos - row_at) / (nb + pause), pair_at = row_at + h * (nb + pause), keys_at = pair_at + pause;
    const int blk0 = max(0, pos - keys_at), blk1 = min(nb, end - keys_at);
    const int lo = kv > 0 ? first_visible_key(kv - 1, a.window, 0) : 0, base_key = at_row.first * kBlock<HD>;
    const int tile0 = (base_key + blk0 * kBlock<HD>) / kKeys<HD> + warp;
    const int tile_end = min((base_key + blk1 * kBlock<HD>) / kKeys<HD>, (kv + kKeys<HD> - 1) / kKeys<HD>);
    const int* bt = a.block_table + (size_t)at_row.table * a.bt_stride;

    // Page of product u of the tile (P16) or of its key lane & 15; -1: nothing of it is seen.
    auto page_of = [&](int tile, int u) -> int {
      const int key = (tile * SUB + u) * kTile + (P16 ? 0 : lane & 15);
      if (tile >= tile_end || ((SUB > 1 || !P16) && key >= kv) || key + (P16 ? kTile - 1 : 0) < lo) return -1;
      return bt[a.ps_shift >= 0 ? key >> a.ps_shift : key / a.page_size];
    };
    auto load_product = [&](int tile, int stage, int u, int page) {
      const uint32_t dst = ring_u32 + stage * S::kStageBytes + u * (2 * kTile * HD);
      const uint32_t scale_to = scales_u32 + ((stage * SUB + u) * 32 + lane) * 4;
      const int first = (tile * SUB + u) * kTile;
      if constexpr (P16) {
        const int slot = a.ps_shift >= 0 ? first & (a.page_size - 1) : first % a.page_size;
        const long unit = (long)page * nkv + h;
        const bool whole = first >= lo && first + kTile <= kv && page >= 0;
        const long off = page >= 0 ? (unit * a.page_size + slot) * HD + lane * 16 : 0;
        const uint8_t *kp = a.k_cache + off, *vp = a.v_cache + off;
        if (whole) {
#pragma unroll
          for (int i = 0; i < CH / 2; ++i) {
            cp_async16(dst + i * 512 + turned_at[i & 1], kp + i * 512, 16);
            cp_async16(dst + kTile * HD + i * 512 + turned_at[i & 1], vp + i * 512, 16);
          }
        } else {
#pragma unroll
          for (int i = 0; i < CH / 2; ++i) {
            const int key = first + (i * 32 + lane) / CH;
            const int bytes = key >= lo && key < kv && page >= 0 ? 16 : 0;
            cp_async16(dst + i * 512 + turned_at[i & 1], bytes ? kp + i * 512 : a.k_cache, bytes);
            cp_async16(dst + kTile * HD + i * 512 + turned_at[i & 1], bytes ? vp + i * 512 : a.v_cache, bytes);
          }
        }
        if (lane < 2) cp_async4(scale_to, (lane ? a.v_scale : a.k_scale) + (page >= 0 ? unit : 0), page >= 0 ? 4 : 0);
      } else {
#pragma unroll
        for (int i = 0; i < CH / 2; ++i) {
          const int part = i * 32 + lane, key = part / CH, abs_key = first + key;
          const int pg = __shfl_sync(0xffffffffu, page, key);
          const int slot = a.ps_shift >= 0 ? abs_key & (a.page_size - 1) : abs_key % a.page_size;
          const size_t off = pg >= 0 ? (((size_t)pg * nkv + h) * a.page_size + slot) * HD + (part % CH) * 16 : 0;
          cp_async16(dst + i * 512 + turned_at[i & 1], a.k_cache + off, pg >= 0 ? 16 : 0);
          cp_async16(dst + kTile * HD + i * 512 + turned_at[i & 1], a.v_cache + off, pg >= 0 ? 16 : 0);
        }
        const float* from = lane < 16 ? a.k_scale : a.v_scale;
        cp_async4(scale_to, from + (page >= 0 ? (size_t)page * nkv + h : 0), page >= 0 ? 4 : 0);
      }
    };

    auto load_tile = [&](int tile, int stage, const int (&page)[SUB]) {
#pragma unroll
      for (int u = 0; u < SUB; ++u) load_product(tile, stage, u, page[u]);
    };

    int page_next[SUB];
    {
      int pg[NS][SUB];
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int u = 0; u < SUB; ++u) pg[i][u] = page_of(tile0 + i * kWarps, u);
#pragma unroll
      for (int i = 0; i < NS - 1; ++i) {
        if (tile0 + i * kWarps < tile_end) load_tile(tile0 + i * kWarps, i, pg[i]);
        cp_commit();
      }
#pragma unroll
      for (int u = 0; u < SUB; ++u) page_next[u] = pg[NS - 1][u];
    }

    // q: lane (g, c) holds numbers c * HD / 4 ... of query g
    uint32_t qb[NT][KS][2];
    float qf[NT][2];                       // scale, log2 e and q's power of two for queries 2c and 2c + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      uint4 raw[HD / 32];
      const bool have = nt * 8 + g < G;
      const uint4* src = reinterpret_cast<const uint4*>(a.q + (size_t)t * a.q_row_stride + (size_t)(h * G + nt * 8 + g) * HD + c * (HD / 4));
      float most = 0.f;
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) raw[i] = have ? src[i] : make_uint4(0, 0, 0, 0);
      auto number = [&](int e) {           // number e of the lane's
        const uint32_t w = reinterpret_cast<const uint32_t*>(raw)[e >> 1];
        return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
      };
#pragma unroll
      for (int e = 0; e < HD / 4; ++e) most = fmaxf(most, fabsf(number(e)));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const int x = min(max((int)(__float_as_uint(most) >> 23) - 127, -100), 127);
      const float up = exp2_int(14 - x);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        qb[nt][s][0] = pack_f16(number(4 * s) * up, number(4 * s + 1) * up);
        qb[nt][s][1] = pack_f16(number(4 * s + 2) * up, number(4 * s + 3) * up);
      }
      const float down = ldexpf(a.scale_log2, x - 14);
      qf[nt][0] = __shfl_sync(0xffffffffu, down, 8 * c);
      qf[nt][1] = __shfl_sync(0xffffffffu, down, 8 * c + 4);
    }

    float o[NT][MT][4], m[NT][2], l[NT][2];
    float mw[NT][2];                       // the second maximum, in log2; o is relative to 2^(mw - kUp)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = mw[nt][0] = mw[nt][1] = kNone;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int j = 0; j < MT; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
    }

    int stage = 0;
    for (int tile = tile0; tile < tile_end; tile += kWarps) {
      const int ahead = tile + (NS - 1) * kWarps;
      if (ahead < tile_end) load_tile(ahead, stage == 0 ? NS - 1 : stage - 1, page_next);
      cp_commit();
#pragma unroll
      for (int u = 0; u < SUB; ++u) page_next[u] = page_of(ahead + kWarps, u);
      cp_wait<NS - 1>();
      __syncwarp();
      const unsigned char* products = ring + stage * S::kStageBytes;
      // of keys g and g + 8 of each product: scores, logarithms of the values' scales, whether they are seen
      float s[SUB][NT][4], lv[SUB][2];
      bool in[SUB][2], grew = false;
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        const unsigned char* kt = products + u * (2 * kTile * HD);
        const float* sc = scales + (stage * SUB + u) * 32;
        float ks[2];
        if constexpr (P16) {
          const float2 x = *reinterpret_cast<const float2*>(sc);
          ks[0] = ks[1] = x.x;
          lv[u][0] = lv[u][1] = log2_fast(x.y);
        } else {
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            ks[y] = sc[g + 8 * y];
            lv[u][y] = log2_fast(sc[16 + g + 8 * y]);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[u][nt][0] = s[u][nt][1] = s[u][nt][2] = s[u][nt][3] = 0.f;
#pragma unroll
        for (int i = 0; i < HD / 64; ++i) {
          const int part = HD == 128 ? ((2 * c + i) ^ g) : (c ^ ((g >> 1) & 3));
          const uint4 w0 = *reinterpret_cast<const uint4*>(kt + g * HD + part * 16);
          const uint4 w1 = *reinterpret_cast<const uint4*>(kt + (g + 8) * HD + part * 16);
          const uint32_t x0[4] = {w0.x, w0.y, w0.z, w0.w}, x1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t a0, a1, a2, a3;
            q8_half4(x0[e], a0, a2);
            q8_half4(x1[e], a1, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16(s[u][nt], a0, a1, a2, a3, qb[nt][4 * i + e][0], qb[nt][4 * i + e][1]);
          }
        }
        const int key0 = (tile * SUB + u) * kTile + g;
#pragma unroll
        for (int y = 0; y < 2; ++y) in[u][y] = key0 + 8 * y >= lo && key0 + 8 * y < kv;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int y = 0; y < 2; ++y) s[u][nt][2 * y + e] = in[u][y] ? s[u][nt][2 * y + e] * (qf[nt][e] * ks[y]) : -INFINITY;
            const float x = fmaxf(s[u][nt][e], s[u][nt][2 + e]), w = P16 ? x + lv[u][0] : fmaxf(s[u][nt][e] + lv[u][0], s[u][nt][2 + e] + lv[u][1]);
            grew |= x > m[nt][e] + kSlack || w > mw[nt][e] + kSlack;
          }
      }
      if (__any_sync(0xffffffffu, grew)) {      // the sums so far follow the maxima
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float f[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = -INFINITY, w = -INFINITY;
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
              x = fmaxf(x, fmaxf(s[u][nt][e], s[u][nt][2 + e]));
              w = fmaxf(w, fmaxf(s[u][nt][e] + lv[u][0], s[u][nt][2 + e] + lv[u][1]));
            }
#pragma unroll
            for (int d = 4; d <= 16; d *= 2) {
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
              w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, d));
            }
            const float mn = fmaxf(m[nt][e], x), wn = fmaxf(mw[nt][e], w);
            l[nt][e] *= exp2_fast(m[nt][e] - mn);
            f[e] = exp2_fast(mw[nt][e] - wn);
            m[nt][e] = mn;
            mw[nt][e] = wn;
          }
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            o[nt][j][0] *= f[0];
            o[nt][j][1] *= f[1];
            o[nt][j][2] *= f[0];
            o[nt][j][3] *= f[1];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            l[nt][e] += exp2_fast(s[u][nt][e] - m[nt][e]) + exp2_fast(s[u][nt][2 + e] - m[nt][e]);
#pragma unroll
            for (int y = 0; y < 2; ++y) w[2 * y + e] = exp2_fast(s[u][nt][2 * y + e] + ((lv[u][y] + kUp) - mw[nt][e]));
          }
          pb[nt][0] = turned(pack_f16(w[0], w[1]));
          pb[nt][1] = turned(pack_f16(w[2], w[3]));
        }
        // values: numbers g * HD / 8 ... of keys 2c, 2c + 1, 2c + 8, 2c + 9; two keys' codes are laced so that a pair of codes is one register of V^T
        const unsigned char* vt = products + u * (2 * kTile * HD) + kTile * HD;
        constexpr int VW = HD / 32;      // words of 4 codes
        uint32_t v[4][VW];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int key = 2 * c + (y & 1) + (y >> 1) * 8;
          if constexpr (HD == 128) {
            const uint4 w = *reinterpret_cast<const uint4*>(vt + key * HD + ((g ^ (key & 7)) * 16));
            v[y][0] = w.x, v[y][1] = w.y, v[y][2] = w.z, v[y][3] = w.w;
          } else {
            const uint2 w = *reinterpret_cast<const uint2*>(vt + key * HD + (((g >> 1) ^ ((key >> 1) & 3)) * 16) + (g & 1) * 8);
            v[y][0] = w.x, v[y][1] = w.y;
          }
        }
#pragma unroll
        for (int w = 0; w < VW; ++w) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t x = __byte_perm(v[0][w], v[1][w], half ? 0x7362 : 0x5140), y = __byte_perm(v[2][w], v[3][w], half ? 0x7362 : 0x5140);
            uint32_t a0, a1, a2, a3;
            q8_half4(x, a0, a1);
            q8_half4(y, a2, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][2 * w + half], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
          }
        }
      }
      __syncwarp();
      stage = stage + 1 == NS ? 0 : stage + 1;
    }
    cp_wait<0>();

    // the four warps' sums: o[nt][j] holds numbers g * HD / 8 + 2j (rows g) and + 1 (rows g + 8) of queries 2c, 2c + 1
    __syncthreads();                                   // the rings are free
    float* mo = reinterpret_cast<float*>(smem);        // [4][NT * 8][kPitch]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = l[nt][e];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        const int query = nt * 8 + 2 * c + e;
        if (g == 0) {
          ml_s[warp][query][0] = m[nt][e];
          ml_s[warp][query][1] = x;
          ml_s[warp][query][2] = mw[nt][e];
        }
        if (query < G) {
          float* dst = mo + (warp * NT * 8 + query) * S::kPitch + 2 * g;
#pragma unroll
          for (int j = 0; j < MT; ++j) *reinterpret_cast<float2*>(dst + 16 * j) = make_float2(o[nt][j][e], o[nt][j][2 + e]);
        }
      }
    }
    __syncthreads();
    const bool whole = blk0 == 0 && blk1 == nb;
    const size_t slot = (size_t)blockIdx.x * 2 + (blk0 == 0);      // a CTA has one cut pair's start and one cut pair's further part at most
    for (int i = tid; i < G * (HD / 4); i += kThreads) {
      const int query = i / (HD / 4), p = i % (HD / 4) * 4;
      float M = kNone, MW = kNone;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        M = fmaxf(M, ml_s[w][query][0]);
        MW = fmaxf(MW, ml_s[w][query][2]);
      }
      float L = 0.f;
      float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = exp2_fast(ml_s[w][query][2] - MW);
        const float4 x = *reinterpret_cast<const float4*>(mo + (w * NT * 8 + query) * S::kPitch + p);
        L += ml_s[w][query][1] * exp2_fast(ml_s[w][query][0] - M);
        O = make_float4(O.x + x.x * f, O.y + x.y * f, O.z + x.z * f, O.w + x.w * f);
      }
      if (whole) {
        finish(t, h * G + query, p, M, L, MW, O, kv <= 0);
      } else {
        *reinterpret_cast<float4*>(a.part_o + (slot * 16 + query) * HD + p) = O;
        if (p == 0) *reinterpret_cast<float4*>(a.part_ml + (slot * 16 + query) * 4) = make_float4(M, L, MW, 0.f);
      }
    }
    if (!whole) {
      // the cuts inside this pair are those farther than `slack` from both of its ends; the piece in front of cut k belongs to CTA k - 1
      const int cut0 = (keys_at + slack) / share + 1, cut1 = (keys_at + nb - slack - 1) / share, pieces = cut1 - cut0 + 2, first_cta = cut0 - 1;
      __syncthreads();
      if (tid == 0) {
        __threadfence();
        int* counter = a.counters + row * nkv + h;
        last_s = atomicAdd(counter, 1) == pieces - 1;
        if (last_s) {
          *counter = 0;
          __threadfence();
        }
      }
      __syncthreads();
      if (last_s) {
        // four numbers a thread; where there are fewer such quads than threads, `sets` of threads take every sets-th piece of a quad and add up their sums
        const int quads = G * (HD / 4), sets = max(1, min(8, kThreads / quads)), set = tid / quads;
        float4* so = reinterpret_cast<float4*>(smem);
        float4* sml = reinterpret_cast<float4*>(smem + kThreads * 16);
        for (int i = sets > 1 ? tid - set * quads : tid; i < quads; i += kThreads) {
          const int query = i / (HD / 4), d = i % (HD / 4) * 4;
          float M = kNone, L = 0.f, MW = kNone;
          float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int k0 = sets > 1 ? set : 0; k0 < (set < sets || sets == 1 ? pieces : 0); k0 += 8 * sets) {      // eight pieces' numbers under way at once
            float4 ml[8], po[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int piece = k0 + k * sets;
              const size_t at = ((size_t)(first_cta + piece) * 2 + (piece == 0)) * 16 + query;
              ml[k] = piece < pieces ? __ldcg(reinterpret_cast<const float4*>(a.part_ml) + at) : make_float4(kNone, 0.f, kNone, 0.f);
              po[k] = piece < pieces ? __ldcg(reinterpret_cast<const float4*>(a.part_o + at * HD + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            float top = M, top_mw = MW;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              top = fmaxf(top, ml[k].x);
              top_mw = fmaxf(top_mw, ml[k].z);
            }
            const float was = exp2_fast(MW - top_mw);
            L *= exp2_fast(M - top);
            O = make_float4(O.x * was, O.y * was, O.z * was, O.w * was);
            M = top;
            MW = top_mw;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float f = exp2_fast(ml[k].z - top_mw);
              L += ml[k].y * exp2_fast(ml[k].x - top);
              O = make_float4(O.x + po[k].x * f, O.y + po[k].y * f, O.z + po[k].z * f, O.w + po[k].w * f);
            }
          }
          if (sets > 1) {
            so[tid] = O;
            sml[tid] = make_float4(M, L, MW, 0.f);
            continue;
          }
          finish(t, h * G + query, d, M, L, MW, O, false);
        }
        if (sets > 1) {
          __syncthreads();
          for (int i = tid; i < quads; i += kThreads) {
            float M = kNone, L = 0.f, MW = kNone;
            float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int k = 0; k < sets; ++k) {
              M = fmaxf(M, sml[k * quads + i].x);
              MW = fmaxf(MW, sml[k * quads + i].z);
            }
            for (int k = 0; k < sets; ++k) {
              const float f = exp2_fast(sml[k * quads + i].z - MW);
              const float4 x = so[k * quads + i];
              L += sml[k * quads + i].y * exp2_fast(sml[k * quads + i].x - M);
              O = make_float4(O.x + x.x * f, O.y + x.y * f, O.z + x.z * f, O.w + x.w * f);
            }
            finish(t, h * G + i / (HD / 4), i % (HD / 4) * 4, M, L, MW, O, false);
          }
        }
      }
    }
    __syncthreads();
    pos = blk1 == nb ? keys_at + nb : end;
  }
}

template <int HD, int NT, bool P16>
__global__ void __launch_bounds__(kThreads, Shape<HD, NT>::kResident) q8_decode_kernel(DecodeArgs a) {
  pdl_launch_dependents();
  if (!a.beside) pdl_wait();
  q8_decode<HD, NT, P16>(a);
  if (a.beside) pdl_wait();      // what comes behind this kernel may rely on the one in front of it too
}

template <int HD, int NT, bool P16>
int launch(const DecodeArgs& a, int ctas, cudaStream_t s) {
  using S = Shape<HD, NT>;
  constexpr size_t merge = (size_t)kWarps * NT * 8 * S::kPitch * 4;
  constexpr size_t smem = S::kSmem > merge ? S::kSmem : merge;
  static SharedLimit limit;
  const cudaError_t raised = limit.raise((const void*)q8_decode_kernel<HD, NT, P16>, smem);
  if (raised != cudaSuccess) return (int)raised;
  // early: one row behind another 10.2 -> 8.8 us, a window's 16.4 -> 15.0, 8 long rows 69.8 -> 68.5 (launched one by one; in a graph there is no difference)
  launch_early(q8_decode_kernel<HD, NT, P16>, dim3(ctas), dim3(kThreads), smem, s, 1, a);
  return launch_status();
}

template <int HD>
int launch_by(const DecodeArgs& a, int ctas, cudaStream_t s) {
  const bool p16 = a.page_size % 16 == 0;
  if (a.nq / a.nkv <= 8) return p16 ? launch<HD, 1, true>(a, ctas, s) : launch<HD, 1, false>(a, ctas, s);
  return p16 ? launch<HD, 2, true>(a, ctas, s) : launch<HD, 2, false>(a, ctas, s);
}

}  // namespace

// Rows with one query; others are left alone.  With positions and row_of_token (int32 [rows]) the rows are the step's tokens, all of them.  Scratch: part_o float32 [ctas * 2 * 16 * hd], part_ml float32 [ctas * 2 * 16 * 4], counters int32
// [rows * nkv], zero before the first launch (the kernel leaves them zero).
// beside: the kernel in front of it on the stream is a prompt kernel launched in stream order that writes none of what this one reads; then this one starts
// as soon as that one's last block has started, on the SMs that it leaves free.  (It starts when all in front of that kernel is done.)
ARLE_API int arle_attention_q8_decode(const void* q, int q_row_stride, void* out, const void* k_cache, const void* v_cache, const float* k_scale,
                                      const float* v_scale, const int* q_indptr, const int* kv_lens, const int* block_table, int bt_stride, float* part_o,
                                      float* part_ml, int* counters, int nq, int nkv, int hd, int page_size, float scale, int window, const float* sinks, int rows,
                                      int ctas, int beside, const int* positions, const int* row_of_token, cudaStream_t s) {
  if (rows <= 0) return 0;
  if (nkv <= 0 || nq <= 0 || nq % nkv || nq / nkv > 16 || page_size <= 0 || ctas <= 0 || (hd != 64 && hd != 128) || q_row_stride % 8) return ARLE_E_UNSUPPORTED;
  int shift = -1;
  if ((page_size & (page_size - 1)) == 0)
    for (shift = 0; (1 << shift) < page_size; ++shift) {}
  const DecodeArgs a{(const __nv_bfloat16*)q, q_row_stride, (__nv_bfloat16*)out, (const uint8_t*)k_cache, (const uint8_t*)v_cache, k_scale, v_scale, q_indptr,
                     kv_lens, block_table, bt_stride, part_o, part_ml, counters, nq, nkv, page_size, shift, window, rows, scale * 1.4426950408889634f, sinks,
                     beside && !(pdl_enabled() & 1), positions, row_of_token};
  return hd == 128 ? launch_by<128>(a, ctas, s) : launch_by<64>(a, ctas, s);
}
