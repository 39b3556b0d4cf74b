// A step's tables from the lengths of its requests: row r of the step is the request in slot slots[r], which holds starts[r] tokens and brings q_lens[r]
// more; page_table[slot] lists its pages.  With held_r = ceil(starts[r] / page_size) and pages_r = ceil((starts[r] + q_lens[r]) / page_size), the row takes
// the next pages_r - held_r of new_pages in the order of rows, and
//     q_indptr = the sums of q_lens in front of each row;   kv_lens[r] = starts[r] + q_lens[r];   page_table[slot][held_r ..] = its new pages
//     block_table[r] = page_table[slot] up to pages_r, -1 behind and for what is no page of the cache;   for token i of row r: position p = starts[r] + i, slot_mapping = page of p * page_size + p % page_size
// Every block sums the lengths of all rows for itself (a few microseconds of latency once, whatever the grid is, where a second launch or a wait for
// another block would cost as much again), then writes its share of the tokens and of the tables' entries.  What is in page_table is read only in front of
// held_r and written only from there on, so blocks do not disturb one another.  Bound by latency, three dependent accesses (lengths, pages, stores): 5.0 us for 8
// rows, 6.5 for 256 with 15,000 tokens and tables of 1,000 pages.
// A step that is not in order (bits of *status below) leaves page_table as it is and an empty step in the outputs: lengths of 0, places and pages of -1.
#include "common.cuh"
using namespace arle;

namespace {

constexpr int kThreads = 512, kMostRows = 4096, kMostSlots = 65536;
enum { kTokens = 1, kSlots = 2, kWidth = 4, kPages = 8, kNegative = 16, kForeign = 32 };

struct StepTables {
  const int *slots, *starts, *q_lens, *new_pages;
  int* page_table;
  int rows, num_new, max_slots, table_width, num_pages, page_size, tokens, width;
  int *q_indptr, *kv_lens, *positions, *row_of_token, *slot_of_token, *slot_mapping, *block_table, *status;
};

__global__ void __launch_bounds__(kThreads) step_tables_kernel(StepTables a) {
  pdl_launch_dependents();
  pdl_wait();
  extern __shared__ int smem[];
  int* until = smem;                  // [rows] tokens up to the row's last
  int* taken = until + a.rows;        // [rows] new pages up to the row's last
  int* begin = taken + a.rows;        // [rows] tokens that it holds
  int* slot = begin + a.rows;         // [rows]
  unsigned* seen = (unsigned*)(slot + a.rows);      // a bit for each slot
  __shared__ long long sums[2][kThreads / 32];
  __shared__ int bad_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, ps = a.page_size;
  for (int i = tid; i < (a.max_slots + 31) / 32; i += kThreads) seen[i] = 0;
  if (tid == 0) bad_s = 0;
  __syncthreads();

  int bad = 0;
  const int each = (a.rows + kThreads - 1) / kThreads, r0 = tid * each, r1 = min(r0 + each, a.rows);
  long long tok = 0, pag = 0;
  for (int r = r0; r < r1; ++r) {
    const int s = a.starts[r], n = a.q_lens[r], at = a.slots[r];
    const long long end = (long long)s + n;
    begin[r] = s;
    slot[r] = at;
    if (s < 0 || n < 0) bad |= kNegative;
    else if (end > (long long)min(a.table_width, a.width) * ps) bad |= kWidth;
    else {
      tok += n;
      pag += (end + ps - 1) / ps - ((long long)s + ps - 1) / ps;
    }
    if (at < 0 || at >= a.max_slots || ((atomicOr(&seen[at >> 5], 1u << (at & 31)) >> (at & 31)) & 1u)) bad |= kSlots;
    until[r] = (int)min(tok, (long long)0x7fffffff);
    taken[r] = (int)min(pag, (long long)0x7fffffff);
  }
  // sums over the threads in front of this one
  long long ti = tok, pi = pag;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, ti, o), y = __shfl_up_sync(0xffffffffu, pi, o);
    if (lane >= o) ti += x, pi += y;
  }
  if (lane == 31) sums[0][warp] = ti, sums[1][warp] = pi;
  __syncthreads();
  long long tw = 0, pw = 0, tall = 0, pall = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) tw += sums[0][w], pw += sums[1][w];
    tall += sums[0][w], pall += sums[1][w];
  }
  if (tall > a.tokens) bad |= kTokens;
  if (pall > a.num_new) bad |= kPages;
  else
    for (int i = tid; i < (int)pall; i += kThreads) {
      const int p = a.new_pages[i];
      if (p < 0 || p >= a.num_pages) bad |= kForeign;
    }
  if (bad) atomicOr(&bad_s, bad);
  tw += ti - tok;
  pw += pi - pag;
  for (int r = r0; r < r1; ++r) until[r] += (int)tw, taken[r] += (int)pw;
  __syncthreads();
  bad = bad_s;
  const int rows = a.rows, g = blockIdx.x * kThreads + tid, all = gridDim.x * kThreads;
  if (g == 0) *a.status = bad;
  if (g == 0) a.q_indptr[0] = 0;
  for (int r = g; r < rows; r += all) {
    a.q_indptr[r + 1] = bad ? 0 : until[r];
    a.kv_lens[r] = bad ? 0 : begin[r] + until[r] - (r ? until[r - 1] : 0);
  }
  const int tokens = bad ? a.tokens : (int)tall;
  for (int t = g; t < tokens; t += all) {
    int lo = 0, pos = 0, sl = 0, place = -1;
    if (!bad) {
      int hi = rows - 1;                       // the first row whose tokens end behind t
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (until[mid] > t) hi = mid;
        else lo = mid + 1;
      }
      const int before = lo ? until[lo - 1] : 0;
      pos = begin[lo] + t - before;
      sl = slot[lo];
      const int j = pos / ps, held = (begin[lo] + ps - 1) / ps;
      const int page = j < held ? a.page_table[(long)sl * a.table_width + j] : a.new_pages[(lo ? taken[lo - 1] : 0) + j - held];
      place = page < 0 || page >= a.num_pages ? -1 : page * ps + pos % ps;
    }
    a.positions[t] = pos;
    a.row_of_token[t] = lo;
    a.slot_of_token[t] = sl;
    a.slot_mapping[t] = place;
  }
  // the tables' entries, a warp for 32 in turn
  const int strips = (a.width + 31) / 32;
  for (long u = (long)blockIdx.x * (kThreads / 32) + warp; u < (long)rows * strips; u += (long)gridDim.x * (kThreads / 32)) {
    const int r = (int)(u / strips), j = (int)(u % strips) * 32 + lane;
    if (j >= a.width) continue;
    int page = -1;
    if (!bad) {
      const int held = (begin[r] + ps - 1) / ps, before = r ? taken[r - 1] : 0, pages = held + taken[r] - before;
      if (j < held) {
        page = a.page_table[(long)slot[r] * a.table_width + j];
        if (page < 0 || page >= a.num_pages) page = -1;      // what reads the table reads the cache there
      } else if (j < pages) {
        page = a.new_pages[before + j - held];
        a.page_table[(long)slot[r] * a.table_width + j] = page;
      }
    }
    a.block_table[(long)r * a.width + j] = page;
  }
}

}  // namespace

// page_table int32 [max_slots, table_width]; block_table int32 [rows, width]; positions and the other tables of tokens hold `tokens` numbers.
ARLE_API int arle_step_tables(const int* slots, const int* starts, const int* q_lens, int rows, const int* new_pages, int num_new, int* page_table, int max_slots,
                              int table_width, int num_pages, int page_size, int* q_indptr, int* kv_lens, int* positions, int* row_of_token, int* slot_of_token,
                              int* slot_mapping, int tokens, int* block_table, int width, int* status, cudaStream_t s) {
  if (rows <= 0 || rows > kMostRows || max_slots <= 0 || max_slots > kMostSlots || page_size <= 0 || num_new < 0 || tokens < 0 || width <= 0 || table_width <= 0 ||
      num_pages < 0 || (long)num_pages * page_size > 0x7fffffffL || (long)width * page_size > 0x7fffffffL)
    return ARLE_E_UNSUPPORTED;
  const size_t smem = (size_t)rows * 16 + (size_t)(max_slots + 31) / 32 * 4;
  static SharedLimit limit;
  if (smem > 48 * 1024) {
    const cudaError_t raised = limit.raise((const void*)step_tables_kernel, (size_t)kMostRows * 16 + kMostSlots / 8);
    if (raised != cudaSuccess) return (int)raised;
  }
  // a block for each 2,048 numbers written, one an SM at most
  const long work = (long)tokens * 4 + (long)rows * width;
  const int blocks = (int)(work <= 2048 ? 1 : work >= 148 * 2048L ? 148 : (work + 2047) / 2048);
  const StepTables a{slots, starts, q_lens, new_pages, page_table, rows, num_new, max_slots, table_width, num_pages, page_size, tokens, width,
                     q_indptr, kv_lens, positions, row_of_token, slot_of_token, slot_mapping, block_table, status};
  launch_kernel(step_tables_kernel, dim3(blocks), dim3(kThreads), smem, s, 1, a);
  return launch_status();
}
