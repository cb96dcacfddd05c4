// The tables of a step -- block table, positions, slots, lengths -- from the requests' lengths, on the GPU.
//
// B requests hold kv[b] tokens in the cache and want new[b] more; the step has room for T new tokens and the free list
// holds page ids from entry `head` on.  With C = ceil(x / block_size):
//   cu[b + 1]     = min(new[0] + .. + new[b], T)                    the step's tokens, request after request
//   acc[b]        = cu[b + 1] - cu[b]                               (requests behind the budget wait)
//   old[b]        = min(C(kv[b]), W),  need[b] = min(C(kv[b] + acc[b]), W) - old[b]        W: width of the table
//   indptr[b + 1] = min(need[0] + .. + need[b], n_free - head)      pages taken, in the order of the free list
//   table[b, j]   = the old entry for j < old[b], free[head + indptr[b] + j - old[b]] for the pages taken, -1 behind them
//   token i of b  : position kv[b] + i - cu[b], slot table[b, position / bs] * bs + position % bs (-1 where no page was left)
//   rows behind the last token: position 0, slot -1
// Everything is integer arithmetic: the result does not depend on the order in which the lanes work.
//
// The two sums saturate at T and at the pages left (min(x + y, cap) is associative for x, y >= 0), so 32 bits hold them
// whatever the lengths.  Up to kFusedBatch requests are one launch: every workgroup makes both sums for itself in LDS
// (they come from L2 after the first) and takes its share of the tokens and of the table; a token finds its request by
// bisection in LDS.  Beyond that a first launch of one workgroup makes the sums and the second reads them from memory.
#include "common.cuh"
#include "launch.h"

namespace xllm_mi355 {

namespace {

// Requests of the one-launch forms: a thread holds a run of one, two or four in registers, and the workgroups are as small
// as that allows, since the barriers of the sums are cheaper (64 decode rows: 3.4 us with 256 threads, 5.8 with 1024; 300
// rows: 3.9 with 256 threads and runs of two, 6.0 with 1024; 1024 rows: 4.3 with 512 and runs of two, 4.9 with 256 and runs
// of four, 6.2 with 1024 and runs of four; 2048 rows: 5.9 with runs of two and 6.7 with runs of four).  Two launches where
// the sums no longer fit LDS (1024 rows: 15 us in two; 4096 rows: 9.2 us in one, 21 in two).
constexpr int kFusedBatch = 4096;        // 3 arrays of up to 16 KB in LDS
constexpr int kSumsThreads = 256;        // of the second of two launches
constexpr int kStepCols = 8;             // table entries of a lane, their loads in flight together

struct StepArgs {
  const int32_t* kv_lens;
  const int32_t* new_lens;
  const int32_t* table_in;
  int32_t* table_out;
  const int32_t* free_pages;
  const int32_t* free_head;   // or null: 0
  int32_t* seq_lens;
  int32_t* cu;
  int64_t* positions;
  int32_t* slots;
  int32_t* indptr;
  int32_t* counters;
  int64_t in_stride, out_stride;
  int batch, width, block_size, bs_shift, budget, n_free;
  int segments;               // of a table row; a wavefront takes one
  int segment_cols;           // at most kWave * kStepCols
};

// Column of a position, and min(C(tokens), W).  (32-bit division: a context and the tokens of a step are below 2^32.)
__device__ __forceinline__ u32 step_column(const StepArgs& a, u32 pos) {
  return a.bs_shift >= 0 ? pos >> a.bs_shift : pos / static_cast<u32>(a.block_size);
}
__device__ __forceinline__ int step_pages(const StepArgs& a, u32 tokens) {
  const u32 full = step_column(a, tokens);
  const u32 n = full + (full * static_cast<u32>(a.block_size) != tokens ? 1u : 0u);
  return static_cast<int>(min(n, static_cast<u32>(a.width)));
}
__device__ __forceinline__ int step_head(const StepArgs& a) {
  return a.free_head != nullptr ? max(0, min(a.free_head[0], a.n_free)) : 0;
}
__device__ __forceinline__ int step_kv(const StepArgs& a, int b) { return max(0, a.kv_lens[b]); }
__device__ __forceinline__ int step_new(const StepArgs& a, int b) { return max(0, min(a.new_lens[b], a.budget)); }

// Saturating exclusive scan of one value per thread; `all` is the sum over the workgroup.  tmp: one word per wavefront.
template <int WAVES>
__device__ __forceinline__ int saturating_scan(int v, int cap, int& all, int* tmp) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  // inside the wavefront by lane moves: rows of 16 lanes first, then the rows' last lanes into the rows behind them
  v = min(v + __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false), cap);   // row_shr:1
  v = min(v + __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false), cap);   // row_shr:2
  v = min(v + __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false), cap);   // row_shr:4
  v = min(v + __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false), cap);   // row_shr:8
  v = min(v + __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false), cap);   // row_bcast:15 into rows 1 and 3
  v = min(v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false), cap);   // row_bcast:31 into rows 2 and 3
  int excl = __builtin_amdgcn_update_dpp(0, v, 0x138, 0xf, 0xf, false);          // wave_shr:1
  __syncthreads();   // (tmp may still be read from the scan before)
  if (lane == kWave - 1) tmp[wave] = v;
  __syncthreads();
  all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const int t = tmp[w];
    if (w < wave) excl = min(excl + t, cap);
    all = min(all + t, cap);
  }
  return excl;
}

// Both sums over the batch into cu[0 .. batch] and indptr[0 .. batch], in global memory and any length of batch.
template <int WAVES>
__device__ __forceinline__ void step_sums(const StepArgs& a, int32_t* cu, int32_t* indptr, int* tmp) {
  const int tid = threadIdx.x;
  const int per = (a.batch + WAVES * kWave - 1) / (WAVES * kWave);
  const int lo = min(a.batch, tid * per), hi = min(a.batch, lo + per);
  const int pages_left = a.n_free - step_head(a);
  int all;
  int sum = 0;
  for (int b = lo; b < hi; ++b) sum = min(sum + step_new(a, b), a.budget);
  int c = saturating_scan<WAVES>(sum, a.budget, all, tmp);
  if (tid == 0) {
    cu[0] = 0;
    indptr[0] = 0;
  }
  const int c0 = c;
  sum = 0;
  for (int b = lo; b < hi; ++b) {
    const int e = min(c + step_new(a, b), a.budget);
    const u32 kv = step_kv(a, b);
    sum = min(sum + (step_pages(a, kv + (e - c)) - step_pages(a, kv)), pages_left);
    cu[b + 1] = e;
    c = e;
  }
  int p = saturating_scan<WAVES>(sum, pages_left, all, tmp);
  c = c0;
  for (int b = lo; b < hi; ++b) {
    const int e = min(c + step_new(a, b), a.budget);
    const u32 kv = step_kv(a, b);
    p = min(p + (step_pages(a, kv + (e - c)) - step_pages(a, kv)), pages_left);
    indptr[b + 1] = p;
    c = e;
  }
  __syncthreads();
}

// The same into LDS, with the pages that each request keeps: a thread's RUN requests stay in registers, so that the
// lengths are read once.
template <int THREADS, int RUN>
__device__ __forceinline__ void step_sums_lds(const StepArgs& a, int32_t* cu, int32_t* indptr, int32_t* old, int* tmp) {
  const int tid = threadIdx.x, lo = tid * RUN;
  int n[RUN], need[RUN];
  u32 kv[RUN];
#pragma unroll
  for (int i = 0; i < RUN; ++i) {
    const bool on = lo + i < a.batch;
    n[i] = on ? step_new(a, lo + i) : 0;
    kv[i] = on ? step_kv(a, lo + i) : 0;
  }
  const int pages_left = a.n_free - step_head(a);
  int all, sum = 0;
#pragma unroll
  for (int i = 0; i < RUN; ++i) sum = min(sum + n[i], a.budget);
  int c = saturating_scan<THREADS / kWave>(sum, a.budget, all, tmp);
  sum = 0;
#pragma unroll
  for (int i = 0; i < RUN; ++i) {
    const int e = min(c + n[i], a.budget);
    const int keep = step_pages(a, kv[i]);
    need[i] = step_pages(a, kv[i] + (e - c)) - keep;
    sum = min(sum + need[i], pages_left);
    if (lo + i < a.batch) {
      cu[lo + i + 1] = e;
      old[lo + i] = keep;
    }
    c = e;
  }
  int p = saturating_scan<THREADS / kWave>(sum, pages_left, all, tmp);
#pragma unroll
  for (int i = 0; i < RUN; ++i) {
    p = min(p + need[i], pages_left);
    if (lo + i < a.batch) indptr[lo + i + 1] = p;
  }
  if (tid == 0) {
    cu[0] = 0;
    indptr[0] = 0;
  }
  __syncthreads();
}

__device__ __forceinline__ int request_of(const int32_t* cu, int batch, int token) {   // cu[b] <= token < cu[b + 1]
  int lo = 0, hi = batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (cu[mid + 1] > token) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// Where entry j of request b's row comes from; null: the entry is -1.
__device__ __forceinline__ const int32_t* step_source(const StepArgs& a, const int32_t* cu, const int32_t* indptr, int b, int j,
                                                      int keep, int head) {
  const int p = indptr[b] + (j - keep);
  const int32_t* src = p < indptr[b + 1] ? a.free_pages + head + p : nullptr;
  return j < keep ? a.table_in + b * a.in_stride + j : src;
}

// What the first workgroup adds: lengths, sums and counters in the caller's arrays.
template <int THREADS>
__device__ __forceinline__ void step_outputs(const StepArgs& a, const int32_t* cu, const int32_t* indptr, bool copy, int* tmp) {
  const int head = step_head(a);
  int lost = 0;   // tokens that no page was left for: those from the end of the request's pages on
  for (int b = threadIdx.x; b < a.batch; b += THREADS) {
    const int64_t kv = step_kv(a, b), total = kv + (cu[b + 1] - cu[b]);
    // (pages that cover the context and the pages taken)
    a.seq_lens[b] = static_cast<int>(total < 0x7fffffffLL ? total : 0x7fffffffLL);
    const int64_t held = static_cast<int64_t>(step_pages(a, static_cast<u32>(kv)) + (indptr[b + 1] - indptr[b])) * a.block_size;
    const int64_t from = held > kv ? held : kv;
    lost += static_cast<int>(total > from ? total - from : 0);
  }
  if (copy)
    for (int b = threadIdx.x; b <= a.batch; b += THREADS) {
      a.cu[b] = cu[b];
      a.indptr[b] = indptr[b];
    }
  int sum;
  saturating_scan<THREADS / kWave>(lost, a.budget, sum, tmp);   // (at most the tokens of the step)
  if (threadIdx.x == 0) {
    a.counters[0] = cu[a.batch];
    a.counters[1] = head + indptr[a.batch];
    a.counters[2] = sum;
  }
}

__global__ __launch_bounds__(1024) void step_sums_kernel(StepArgs a) {
  __shared__ int tmp[16];
  step_sums<16>(a, a.cu, a.indptr, tmp);
  __threadfence_block();
  __syncthreads();
  step_outputs<1024>(a, a.cu, a.indptr, false, tmp);
}

// Pieces of the tokens, a token per thread (with four per thread 22077 tokens of 134 requests took 5.9 us, now 3.6), then
// those of the table.
template <int THREADS>
__host__ __device__ __forceinline__ int token_pieces(const StepArgs& a) {
  return static_cast<int>((static_cast<int64_t>(a.budget) + THREADS - 1) / THREADS);
}
template <int THREADS>
__host__ __device__ __forceinline__ int64_t step_pieces(const StepArgs& a) {
  const int64_t units = static_cast<int64_t>(a.batch) * a.segments;
  return token_pieces<THREADS>(a) + (units + THREADS / kWave - 1) / (THREADS / kWave);
}

// One piece of the tokens, or of the table.  OLD: the pages that the requests keep are in `old`.
template <int THREADS, bool OLD>
__device__ __forceinline__ void step_piece(const StepArgs& a, int64_t piece, const int32_t* cu, const int32_t* indptr,
                                           const int32_t* old, int head) {
  const int tid = threadIdx.x;
  auto kept = [&](int b) { return OLD ? old[b] : step_pages(a, step_kv(a, b)); };
  const int of_tokens = token_pieces<THREADS>(a);
  if (piece < of_tokens) {
    const int64_t i = piece * THREADS + tid;
    if (i >= a.budget) return;
    int64_t pos = 0;
    int slot = -1;
    if (i < cu[a.batch]) {
      const int token = static_cast<int>(i), b = request_of(cu, a.batch, token);
      const u32 kv = step_kv(a, b);
      pos = kv + static_cast<u32>(token - cu[b]);
      const u32 col = step_column(a, static_cast<u32>(pos));
      if (col < static_cast<u32>(a.width)) {
        const int32_t* src = step_source(a, cu, indptr, b, static_cast<int>(col), kept(b), head);
        const int64_t page = src != nullptr ? *src : -1;
        const int64_t s = page * a.block_size + (pos - static_cast<int64_t>(col) * a.block_size);
        if (page >= 0 && s <= 0x7fffffffLL) slot = static_cast<int>(s);
      }
    }
    a.positions[i] = pos;
    a.slots[i] = slot;
    return;
  }
  // A wavefront per segment of a row: the request and its pages are the same in all lanes, which leaves a comparison and
  // a load per entry (with a lane per entry of the flat table the divisions and look-ups were most of the launch: 13.6 us
  // for 2 M entries).  The lanes' loads are issued before the first is used: an entry without a source reads the row's
  // first one, so that no load hangs off a branch.
  const bool in_place = a.table_in == a.table_out;
  const int64_t unit = (piece - of_tokens) * (THREADS / kWave) + __builtin_amdgcn_readfirstlane(tid / kWave);
  const int lane = tid & (kWave - 1);
  const int64_t row_of = unit <= 0x7fffffffLL ? static_cast<u32>(unit) / static_cast<u32>(a.segments) : unit / a.segments;
  if (row_of >= a.batch) return;
  const int b = static_cast<int>(row_of);
  const int c0 = static_cast<int>(unit - row_of * a.segments) * a.segment_cols, c1 = min(a.width, c0 + a.segment_cols);
  const int keep = __builtin_amdgcn_readfirstlane(kept(b));
  const int first = __builtin_amdgcn_readfirstlane(indptr[b]);
  const int end = keep + __builtin_amdgcn_readfirstlane(indptr[b + 1]) - first;   // entries from here on are -1
  const int32_t* row = a.table_in + b * a.in_stride;
  const int32_t* fresh = a.free_pages + head + first - keep;
  int32_t* out = a.table_out + b * a.out_stride;
  int32_t value[kStepCols];
#pragma unroll
  for (int k = 0; k < kStepCols; ++k) {
    const int j = c0 + k * kWave + lane;
    const bool old = j < keep && j < c1 && !in_place;
    const int32_t* src = old ? row + j : row;
    src = j >= keep && j < end && j < c1 ? fresh + j : src;
    value[k] = c0 + k * kWave < min(c1, end) ? *src : -1;
  }
#pragma unroll
  for (int k = 0; k < kStepCols; ++k) {
    const int j = c0 + k * kWave + lane;
    if (j < c1 && !(in_place && j < keep)) out[j] = j < end ? value[k] : -1;
  }
}

template <int THREADS, int RUN>
__global__ __launch_bounds__(THREADS) void step_tables_kernel(StepArgs a) {
  extern __shared__ int32_t lds[];
  __shared__ int tmp[THREADS / kWave];
  int32_t* cu = lds;
  int32_t* indptr = cu + a.batch + 1;
  int32_t* old = indptr + a.batch + 1;
  step_sums_lds<THREADS, RUN>(a, cu, indptr, old, tmp);
  if (blockIdx.x == 0) {   // (a workgroup of its own for the per-request outputs: with pieces on top it would end last)
    step_outputs<THREADS>(a, cu, indptr, true, tmp);
    return;
  }
  const int head = step_head(a);
  const int64_t n = step_pieces<THREADS>(a);
  for (int64_t p = blockIdx.x - 1; p < n; p += gridDim.x - 1) step_piece<THREADS, true>(a, p, cu, indptr, old, head);
}

template <int THREADS, int RUN>
void launch_step_tables(const StepArgs& a, int64_t most, hipStream_t stream) {
  const int64_t n = step_pieces<THREADS>(a) + 1;
  step_tables_kernel<THREADS, RUN><<<dim3(static_cast<unsigned>(n < most ? n : most)), THREADS,
                                     static_cast<size_t>(3 * a.batch + 2) * 4, stream>>>(a);
}

__global__ __launch_bounds__(kSumsThreads) void step_tables_from_sums_kernel(StepArgs a) {
  const int head = step_head(a);
  const int64_t n = step_pieces<kSumsThreads>(a);
  for (int64_t p = blockIdx.x; p < n; p += gridDim.x)
    step_piece<kSumsThreads, false>(a, p, a.cu, a.indptr, nullptr, head);
}

}  // namespace

int build_step_tables(const int32_t* kv_lens, const int32_t* new_lens, const int32_t* block_table_in,
                      int64_t in_stride, int32_t* block_table_out, int64_t out_stride, int64_t table_width,
                      const int32_t* free_pages, int64_t n_free, const int32_t* free_head, int32_t* seq_lens,
                      int32_t* cu_new, int64_t* positions, int32_t* slots, int32_t* new_page_indptr,
                      int32_t* counters, int64_t batch, int64_t block_size, int64_t max_new_tokens,
                      hipStream_t stream) {
  if (batch == 0) return XLLM_MI355_OK;
  if (kv_lens == nullptr || new_lens == nullptr || block_table_in == nullptr || block_table_out == nullptr ||
      (free_pages == nullptr && n_free != 0) || seq_lens == nullptr || cu_new == nullptr || new_page_indptr == nullptr ||
      counters == nullptr || (max_new_tokens > 0 && (positions == nullptr || slots == nullptr)))
    return XLLM_MI355_EINVAL;
  if (batch < 0 || block_size <= 0 || table_width <= 0 || n_free < 0 || max_new_tokens < 0 || in_stride < table_width ||
      out_stride < table_width)
    return XLLM_MI355_EINVAL;
  constexpr int64_t kLimit = (1LL << 30) - 1;   // the sum of two stays inside 32 bits
  if (max_new_tokens > kLimit || n_free > kLimit || table_width > kLimit || block_size > kLimit || batch > (1LL << 20))
    return XLLM_MI355_ESHAPE;
  // No output meets an input or another output, but for the table in place, entry for entry.
  {
    const bool in_place = block_table_in == block_table_out;
    if (in_place && in_stride != out_stride) return XLLM_MI355_EINVAL;
    const Span read[5] = {Span(kv_lens, batch * 4), Span(new_lens, batch * 4), Span(free_pages, n_free * 4),
                          Span(free_head, 4), span_of(block_table_in, batch, in_stride, 1, 0, table_width, 4)};
    const Span written[7] = {span_of(block_table_out, batch, out_stride, 1, 0, table_width, 4), Span(seq_lens, batch * 4),
                             Span(cu_new, batch * 4 + 4), Span(positions, max_new_tokens * 8), Span(slots, max_new_tokens * 4),
                             Span(new_page_indptr, batch * 4 + 4), Span(counters, 12)};
    for (int i = 0; i < 7; ++i) {
      for (int j = 0; j < 5; ++j)
        if (written[i].meets(read[j]) && !(in_place && i == 0 && j == 4)) return XLLM_MI355_EINVAL;
      for (int j = 0; j < i; ++j)
        if (written[i].meets(written[j])) return XLLM_MI355_EINVAL;
    }
  }
  StepArgs a = {};
  a.kv_lens = kv_lens;
  a.new_lens = new_lens;
  a.table_in = block_table_in;
  a.table_out = block_table_out;
  a.free_pages = free_pages;
  a.free_head = free_head;
  a.seq_lens = seq_lens;
  a.cu = cu_new;
  a.positions = positions;
  a.slots = slots;
  a.indptr = new_page_indptr;
  a.counters = counters;
  a.in_stride = in_stride;
  a.out_stride = out_stride;
  a.batch = static_cast<int>(batch);
  a.width = static_cast<int>(table_width);
  a.block_size = static_cast<int>(block_size);
  a.bs_shift = -1;
  for (int s = 0; s < 31; ++s)
    if ((1LL << s) == block_size) a.bs_shift = s;
  a.budget = static_cast<int>(max_new_tokens);
  a.n_free = static_cast<int>(n_free);
  a.segments = static_cast<int>((table_width + kWave * kStepCols - 1) / (kWave * kStepCols));
  a.segment_cols = static_cast<int>((table_width + a.segments - 1) / a.segments);
  // Every workgroup of the one-launch forms makes the sums for itself, so there are no more of them than run at once: 2048
  // threads per CU, and one workgroup per CU of 1024 (2048 requests, 2 M table entries, 65536 tokens: 8.7 us; with two per
  // CU 11 us; with one per piece of work 91 us).
  const int64_t cus = device_cu_count();
  if (batch <= kFusedBatch) {
    if (batch <= 256) launch_step_tables<256, 1>(a, 8 * cus, stream);
    else if (batch <= 512) launch_step_tables<256, 2>(a, 8 * cus, stream);
    else if (batch <= 1024) launch_step_tables<512, 2>(a, 4 * cus, stream);
    else if (batch <= 2048) launch_step_tables<1024, 2>(a, cus, stream);
    else launch_step_tables<1024, 4>(a, cus, stream);
    return static_cast<int>(hipGetLastError());
  }
  step_sums_kernel<<<1, 1024, 0, stream>>>(a);
  const int rc = static_cast<int>(hipGetLastError());
  if (rc != 0) return rc;
  const int64_t pieces = step_pieces<kSumsThreads>(a), most = 16 * cus;
  step_tables_from_sums_kernel<<<dim3(static_cast<unsigned>(pieces < most ? pieces : most)), kSumsThreads, 0, stream>>>(a);
  return static_cast<int>(hipGetLastError());
}

}  // namespace xllm_mi355
