// Differential attention of one new token per sequence over paged keys and values, for gfx950.
//
//   S_m[t]  = scale * q[b, 2h + m] . K[t, 2j + m]          m = 0, 1 (the two maps of head h), j = h / group
//   o       = (softmax(S_0) - lambda[b, h] * softmax(S_1)) . V[:, j]        V rows of 2 D values
//   out     = out_scale * norm_w * o / sqrt(mean(o^2) + eps)                (norm_w null: out = out_scale * o)
//
// The KV heads of a token lie pair after pair, so the two key rows of a pair are one run of 2 D values, of the same
// size and at the same place in the key cache as the value row in the value cache: one address per token serves both.
// A decode step reads every key and value once for a few operations per byte, so the kernel is HBM bound and is built
// to keep bytes in flight; both maps are taken in the one pass over the rows (two ordinary decodes would read V twice).
//
// Schedule.  The context of every (sequence, head block) is cut into stages of 16 tokens.  A worker is one wavefront, four
// or eight to a workgroup, one workgroup per CU; a team is the 4, 2 or 1 workers of a workgroup (as the head blocks divide) that
// walk the same stages of adjacent head blocks side by side, so that what they ask for at a time is one run of memory: a
// token's pairs lie next to each other.  The stages of the batch form one list ordered (sequence, group of head blocks,
// stage); every team streams an equal range of it, whatever the mix of lengths, and its workers meet neither each other
// nor other teams after the common prefix sum of the lengths.  A range that holds a whole context writes the output rows,
// a part of a context goes to the workspace as (o, max, sum) in fp32 and diff_merge_kernel joins the parts.
//
// Data path.  Rows travel from global memory straight into a ring of the worker's own LDS (two stages: 32 KB for 512-byte
// rows, 16 KB for 256-byte rows, of which a CU has twice the workers), and the place of a stage's keys is filled again as soon as they are in registers, the
// place of its values likewise.  Page-table entries take the same path two ring lengths ahead, so that no load of the
// loop waits in a register (such a wait would also wait for every younger row in flight: the counter is in order).
//   S^T[token, column] = K[token, dims] . Q^T        v_mfma_f32_16x16x32, K read from LDS, Q^T in registers
//   O^T[dim, column]  += V^T[dim, token] . P^T       v_mfma_f32_16x16x32, V^T by the transposing LDS read, P^T straight
//                                                    from the accumulators of S^T
// The 16 columns hold both maps of up to eight heads (map 0 in columns 0-7, map 1 in 8-15); both maps' keys are multiplied
// with all of them, and a column keeps the scores of its own.  Groups of more than eight heads take two
// blocks of 16 columns, one per map, so that rows are still read once for sixteen heads.
// P is rounded to the 16-bit type in two parts, p = hi + lo, and both go through the matrix cores: the difference of the
// maps can cancel most of o, which would leave the rounding of a single 16-bit P as the error of what remains (the norm
// scales it up).  It is free: a stage's 16 tokens fill half the depth of a 16x16x32 MFMA, and the other half takes the same
// values against lo.  What the parts leave over: of bf16 2^-16 of p.  Of fp16, whose values end at 2^-25, 2^-22 of p and
// 2^-25 absolute; so its probabilities are held against a maximum 14 powers of two lower and reach 2^14 to 2^15
// (DiffProbs), which leaves 2^-39 of the largest: a token 27 nats below the first one is lost from o, one 18 below keeps
// 12 bits.  (Held against the maximum itself, where fp16's upper half lies idle, a context whose first token has no value
// of its own -- a sink -- lost 42 % of its result at 18 nats.)
// Softmax statistics, sums and the norm are in fp32.
//
// Measured (bf16, 128-dim maps, 16-bit caches): 64 sequences of 0.5k to 4k tokens, 4 pairs, 16 heads (568 MB) 89 us and 6 us
// of merge, 6.4 TB/s in the decode kernel; 256 sequences of 1k to 8k tokens, 32 heads (4.66 GB) 700 us and 11 us, 6.65 TB/s,
// where a plain read of as many bytes runs at 7.05 TB/s.  4 sequences of up to 512 tokens: 5.8 us and 4.7 us, all latency (the
// chain lengths -> page entries -> rows, then the merge's prefix -> parts).  Groups of sixteen heads (64 sequences, 64 heads):
// 5.0 TB/s, bound by the moves between accumulation and ordinary registers around their 128 accumulators.
#include "common.cuh"
#include "launch.h"

namespace xllm_mi355 {

namespace {

constexpr int kDiffTokens = 16;               // tokens of a stage
constexpr int kDiffRings = 131072;            // ring bytes of a workgroup
constexpr int kDiffMaxBatch = 1024;           // sequences per launch (their prefix and lengths lie in LDS)
// A team takes at least two stages once a quarter of the teams are busy and no team has to take two contexts for it; below
// that one, since a short list is all latency (117 sequences of 10 tokens, 8 pairs: 9.1 us, with two contexts a team 12.3).
// (One, two, four at least: 4 contexts of up to 512 tokens 11.4, 12.5, 14.9 us; one of 100 tokens 13.0, 15.9, 21.6 us; one
// of 4000 tokens, which is then in 250, 125 or 62 parts, 24.4, 20.3, 21.7 us.)
constexpr int kDiffMinStages = 2;
// Output rows up to which the parts of a row are joined by a workgroup of 16 or 8 wavefronts, and of 4 (one wavefront beyond).
// 1024 rows of 5 parts: 6 us with 4 and with one; 8192 rows of 2 parts: 34 us with 4, 14 us with one.  Up to 256 rows: 16
// wavefronts where a row may have more than kDiffManyParts parts (16 rows of 250 parts: 12.5 us with 16, 15 with 8, 30 with
// 4), 8 otherwise (32 rows of up to 16 parts: 4.4 us with 8 and 5.0 with 16; 256 rows of some 10: 5.2 and 6.0).
constexpr int64_t kDiffSplit8 = 256, kDiffSplit4 = 2048, kDiffManyParts = 64;
// Output rows from which the parts of 256-dim rows are stored past the caches (up to eight heads per pair).  In a row of
// launches, the merge reading them right behind: 256 sequences x 16 heads of 1k to 8k tokens 695 us and 715 through the
// caches, 128 x 32 heads 364 and 373, 512 x 16 heads of 0.5k to 2k 407 and 419; but 64 x 16 heads 98.5 and 97, 1 x 8 heads of
// 32k 41.4 and 39.2, groups of sixteen (64 x 64 heads) 142 and 137, rows of 128 dims (512 x 32 heads) 246 and 243.
constexpr int64_t kDiffStreamRows = 4096;

// The running maximum against which a worker holds its probabilities (log2 units): it is set kLift below the largest score
// and moves when a score passes it by more than kLift + kSlack, so that e = exp2(s - m) stays below 2^(kLift + kSlack).
// bf16 has fp32's range, and a wide slack keeps the moves rare.  fp16 ends at 2^16: the slack is what it can be with the
// probabilities at the top of its range.  The moves that this adds (some two a context) are not seen in the times but for the
// shape with the most accumulators (64 sequences, 64 heads of 128 dims, groups of sixteen: 133.0 us in fp16, 128.0 in bf16).
template <typename QT>
struct DiffProbs {
  static constexpr float kLift = QT::kIsBf16 ? 0.0f : 14.0f;
  static constexpr float kSlack = QT::kIsBf16 ? 8.0f : 1.0f;
};

typedef __attribute__((address_space(3))) s16x4 diff_lds_s16x4;

struct DiffArgs {
  const char* q;
  const char* k_cache;
  const char* v_cache;
  char* out;
  const int32_t* block_table;
  const int32_t* seq_lens;
  const float* lambda;
  const char* norm_w;
  int* ws_prefix;       // [batch + 1], written by workgroup 0 for the merge
  float* ws_o;          // [2 * workers][columns][2 D]
  float* ws_ml;         // [2 * workers][columns][2]: running maximum (log2 units, see DiffProbs), sum
  int64_t table_stride;
  int64_t q_stride_bytes;
  int64_t out_stride_bytes;
  int64_t row_bytes;    // bytes of a token in either cache
  int64_t lambda_batch_stride;
  int64_t lambda_head_stride;
  int batch;
  int n_heads;          // differential heads
  int n_pairs;          // KV pairs
  int group;            // heads per pair
  int hb_per_pair;      // head blocks per pair
  int block_size;
  int bs_shift;         // log2(block_size) or -1
  int num_blocks;
  int max_len;          // what the table can hold
  int window_left;
  int n_workers;
  int team_shift;       // log2 of the workers of a team (1, 2 or 4)
  // The list in two pools, 9 : 8, one for the workgroups of even number and one for the others (0: one list).  On the full
  // chip (256 CUs, workgroup i on XCD i % 8) the odd XCDs stream slower with equal shares: 9 : 8 takes 4 % off the launch
  // (256 sequences: 771 -> 742 us; 16 : 15 740, 16 : 17 769).  A tuned share and no more: every device computes the same.
  int pools;
  int stream_parts;     // 1: partial rows are stored past the caches
  float scale_log2;
  float eps;
  float out_scale;
};

__device__ __forceinline__ int diff_len(const DiffArgs& a, int b) { return max(0, min(a.seq_lens[b], a.max_len)); }
__device__ __forceinline__ int diff_first(const DiffArgs& a, int L) {
  return a.window_left < 0 ? 0 : max(0, L - 1 - a.window_left);
}
__device__ __forceinline__ int diff_stages(const DiffArgs& a, int L) {
  return L > 0 ? (L + kDiffTokens - 1) / kDiffTokens - diff_first(a, L) / kDiffTokens : 0;
}
// How the list is dealt: stages in equal ranges, the first `rem` of them one longer.  With two pools (below) the first
// `half` teams share the stages before `cut` that way, the others those behind it.
// (Divisions are what this is careful with: 40 dependent instructions each in 32 bits, a hundred in 64, all of them before
// a wavefront's first load.)
__device__ __forceinline__ int64_t diff_div(int64_t x, int64_t y) {
  return ((x | y) >> 32) == 0 ? static_cast<u32>(x) / static_cast<u32>(y) : x / y;
}
struct DiffShare {   // `n` ranges over `total` stages
  int64_t per, rem;
  __device__ __forceinline__ DiffShare(int64_t total, int n) : per(diff_div(total, n)), rem(total - per * n) {}
  __device__ __forceinline__ int64_t start(int w) const { return w * per + (w < rem ? w : rem); }
  __device__ __forceinline__ int owner(int64_t id) const {
    const int64_t big = rem * (per + 1);   // (stages of the longer ranges; per is positive where they end before id)
    return static_cast<int>(id < big ? diff_div(id, per + 1) : rem + diff_div(id - big, per));
  }
};
constexpr int kPoolEven = 9, kPoolOdd = 8;
struct DiffDeal {
  int64_t total, cut;
  int used, half;
};
__device__ __forceinline__ DiffDeal diff_deal(const DiffArgs& a, int64_t total) {
  DiffDeal d;
  d.total = total;
  const int most = a.n_workers >> a.team_shift;
  int64_t n = total / kDiffMinStages, floor = static_cast<int64_t>(a.batch) * ((a.n_pairs * a.hb_per_pair) >> a.team_shift);
  if (floor < most / 4) floor = most / 4;
  if (n < floor) n = total < floor ? total : floor;
  d.used = static_cast<int>(n < most ? n : most);
  const bool pools = a.pools != 0 && d.used == most;
  d.half = pools ? most / 2 : 0;
  d.cut = pools ? total * kPoolEven / (kPoolEven + kPoolOdd) : 0;
  return d;
}
// The range [begin, end) of team w.
__device__ __forceinline__ void diff_range(const DiffDeal& d, int w, int64_t& begin, int64_t& end) {
  const bool second = w >= d.half;
  const int n = d.half == 0 ? d.used : second ? d.used - d.half : d.half;
  const int64_t base = second ? d.cut : 0;
  const DiffShare share((second ? d.total : d.cut) - base, n);
  const int q = second ? w - d.half : w;
  begin = base + share.start(q);
  end = base + share.start(q + 1);
}
// The team whose range holds stage `id`, and where that range begins.
__device__ __forceinline__ int diff_team_of(const DiffDeal& d, int64_t id, int64_t& begin) {
  const bool second = id >= d.cut;
  const int n = d.half == 0 ? d.used : second ? d.used - d.half : d.half;
  const int64_t base = second ? d.cut : 0;
  const DiffShare share((second ? d.total : d.cut) - base, n);
  const int q = share.owner(id - base);
  begin = base + share.start(q);
  return q + (second ? d.half : 0);
}

__device__ __forceinline__ void diff_dma16(const char* p, u32 lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"s"(lds), "v"(p) : "memory");
}
__device__ __forceinline__ void diff_dma4(const int32_t* p, u32 lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(p) : "memory");
}
template <int N>
__device__ __forceinline__ void diff_wait_vm() {
  static_assert(N >= 0 && N < 64, "range of the counter");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void diff_wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

__device__ __forceinline__ float diff_rows_max(float x) {  // over lanes l, l ^ 16, l ^ 32, l ^ 48
  auto t = __builtin_amdgcn_permlane16_swap(as_u32(x), as_u32(x), false, false);
  x = fmaxf(as_f32(t[0]), as_f32(t[1]));
  auto u = __builtin_amdgcn_permlane32_swap(as_u32(x), as_u32(x), false, false);
  return fmaxf(as_f32(u[0]), as_f32(u[1]));
}
__device__ __forceinline__ float diff_rows_sum(float x) {
  auto t = __builtin_amdgcn_permlane16_swap(as_u32(x), as_u32(x), false, false);
  x = as_f32(t[0]) + as_f32(t[1]);
  auto u = __builtin_amdgcn_permlane32_swap(as_u32(x), as_u32(x), false, false);
  return as_f32(u[0]) + as_f32(u[1]);
}

// v0 - lambda v1 with both maps' results rounded alike: left to itself the compiler fuses the first one's normalisation
// into the subtraction, and two equal maps with lambda = 1 leave its rounding behind instead of zero.
__device__ __forceinline__ float diff_of(float v0, float lam, float v1) {
#pragma clang fp contract(off)
  const float t = lam * v1;
  return v0 - t;
}

// A stage of the list.  Every field is the same in all lanes.
struct DiffCursor {
  int b, hg, st, n;    // sequence, group of head blocks, stage, stages of the context
  int L, lo;           // context length, first attended token
  int pair, head0;     // the worker's KV pair and first head
};

template <int D, int NB>
struct DiffShape {
  // One worker per SIMD for rows of 512 bytes, two for rows of 256, which bring half the bytes for the same instructions.
  // 64 sequences of 1k to 8k tokens over 4 pairs of 64-dim maps: 99 us with two and 102 with one for 16 heads, 111 and 124
  // for 64 heads; of 128-dim maps and 16 heads: 97 and 96 us (0.5k to 4k tokens), where the loop waits for memory and not
  // for its instructions (without its P.V products it takes 2 % less).
  static constexpr int kWaves = D == 64 ? 8 : 4;
  // Registers as if two wavefronts shared a SIMD, which they do or could, but for the shape whose accumulators alone are
  // 128: with all 512 the compiler keeps accumulators in accumulation registers and copies them to ordinary ones and back
  // around every product, a third of the loop's instructions.
  static constexpr int kPerSimd = D == 128 && NB == 2 ? 1 : 2;
  static constexpr int kThreads = kWaves * kWave;
  static constexpr int kRing = kDiffRings / kWaves;         // ring bytes of a worker
  static constexpr int kRow = 4 * D;                       // bytes of a pair's row
  static constexpr int kChunks = kRow / 16;                // 16-byte chunks of a row
  static constexpr int kRowsPerLoad = kWave / kChunks;
  static constexpr int kLoads = kDiffTokens / kRowsPerLoad; // load instructions of a stage's keys, and of its values
  static constexpr int kTile = kDiffTokens * kRow;         // bytes of a stage's keys
  static constexpr int kStages = kRing / (2 * kTile);  // ring length
  static constexpr int kPageSlots = 2 * kStages;           // page-table entries are fetched two ring lengths ahead
  static constexpr int kCols = 16 * NB;
  static constexpr int kHeads = NB == 1 ? 8 : 16;          // heads of a head block
  // Query rows and lambdas of a context take the LDS path too.  Those of sixteen heads do not fit beside the rings: they
  // are fetched into registers, which waits for all rows in flight at every change of context.
  static constexpr bool kQueryLds = NB == 1;
  static constexpr int kQueryBytes = kQueryLds ? kHeads * kRow : 0;
  static constexpr int kQueryLoads = kQueryBytes / (kWave * 16);
  // LDS: rings | page entries [waves][kPageSlots][16] | queries [waves] | lambdas [waves][64] | norm weights | scan scratch
  //      [8] | lengths [batch] | prefix [batch + 1]
  static constexpr int kPageOff = kDiffRings;
  static constexpr int kQueryOff = kPageOff + kWaves * kPageSlots * 64;
  static constexpr int kLambdaOff = kQueryOff + kWaves * kQueryBytes;
  static constexpr int kNormOff = kLambdaOff + kWaves * kWave * 4;
  static constexpr int kTmpOff = kNormOff + 4 * D;
  static constexpr int kLensOff = kTmpOff + 32;
  static constexpr size_t lds_bytes(int batch) { return kLensOff + static_cast<size_t>(2 * batch + 1) * 4; }
  static_assert(lds_bytes(kDiffMaxBatch) <= 163840, "LDS of a CU");
};

// One head's finished row: o0 and o1 are the normalised results of the two maps for the lane's dims
// 16 mb + 4 (lane / 16) + r; norm: the weights in LDS.  All four lanes of a head (l, l ^ 16, l ^ 32, l ^ 48) call it together.
template <typename QT, int MB>
__device__ __forceinline__ void diff_store_row(const DiffArgs& a, const char* norm, const f32x4 (&o)[MB], int b, int head, bool on, int g) {
  float ss = 0.0f;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int r = 0; r < 4; ++r) ss += o[mb][r] * o[mb][r];
  ss = diff_rows_sum(ss);
  float f = a.out_scale;
  if (a.norm_w != nullptr) f *= 1.0f / __builtin_sqrtf(ss / static_cast<float>(MB * 16) + a.eps);
  if (!on) return;
  char* row = a.out + b * a.out_stride_bytes + static_cast<int64_t>(head) * MB * 32;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    f32x4 w = {1.0f, 1.0f, 1.0f, 1.0f};
    if (a.norm_w != nullptr) {
      const u32x2 x = *reinterpret_cast<const u32x2*>(norm + (mb * 16 + 4 * g) * 2);
      w = f32x4{QT::lo(x[0]), QT::hi(x[0]), QT::lo(x[1]), QT::hi(x[1])};
    }
    const u32x2 y = {QT::pack(o[mb][0] * f * w[0], o[mb][1] * f * w[1]), QT::pack(o[mb][2] * f * w[2], o[mb][3] * f * w[3])};
    *reinterpret_cast<u32x2*>(row + (mb * 16 + 4 * g) * 2) = y;
  }
}

template <typename QT, int D, int NB>
__global__ __launch_bounds__((DiffShape<D, NB>::kThreads), (DiffShape<D, NB>::kPerSimd)) void diff_decode_kernel(DiffArgs a) {
  using S = DiffShape<D, NB>;
  constexpr int kThreads = S::kThreads;
  constexpr int KS = D / 32;       // k-steps of a map's scores
  constexpr int MB = 2 * D / 16;   // dim blocks of the output
  constexpr int NS = S::kStages;
  constexpr int NL = S::kLoads;
  constexpr float kTop = DiffProbs<QT>::kLift + DiffProbs<QT>::kSlack;
  constexpr int kStageOps = 1 + 2 * NL;   // vector memory operations of a stage: page entries, keys, values
  static_assert(NS >= 2, "the wait for query rows leaves one younger stage in flight");

  extern __shared__ __align__(16) char smem[];
  int* tmp = reinterpret_cast<int*>(smem + S::kTmpOff);
  int* lens = reinterpret_cast<int*>(smem + S::kLensOff);
  int* prefix = lens + a.batch;
  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, g = lane >> 4;
  const int n_hg = (a.n_pairs * a.hb_per_pair) >> a.team_shift;

  // ---- norm weights, lengths and the exclusive prefix sum of the stages
  if (a.norm_w != nullptr)
    for (int i = tid; i < D; i += kThreads)
      reinterpret_cast<u32*>(smem + S::kNormOff)[i] = reinterpret_cast<const u32*>(a.norm_w)[i];
  {
    const int per = (a.batch + kThreads - 1) / kThreads;
    const int lo = min(a.batch, tid * per), hi = min(a.batch, lo + per);
    int local = 0;
    for (int b = lo; b < hi; ++b) {
      const int L = diff_len(a, b);
      lens[b] = L;
      local += diff_stages(a, L);
    }
    int incl = local;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int t = __shfl_up(incl, d, kWave);
      if (lane >= d) incl += t;
    }
    if (lane == kWave - 1) tmp[wave] = incl;
    __syncthreads();
    int excl = incl - local;
    for (int w = 0; w < wave; ++w) excl += tmp[w];
    for (int b = lo; b < hi; ++b) {
      prefix[b] = excl;
      excl += diff_stages(a, lens[b]);
    }
    if (tid == kThreads - 1) prefix[a.batch] = excl;   // (an empty slice leaves the total as it came in)
    __syncthreads();
  }
  if (blockIdx.x == 0)
    for (int b = tid; b <= a.batch; b += kThreads) a.ws_prefix[b] = prefix[b];

  const int64_t total = static_cast<int64_t>(prefix[a.batch]) * n_hg;
  if (total == 0) return;
  const DiffDeal deal = diff_deal(a, total);
  // neighbours in the list sit on different CUs, so that a short list still spreads over the chip
  const int member = wave & ((1 << a.team_shift) - 1), set = wave >> a.team_shift;
  const int team = deal.half == 0 ? set * gridDim.x + blockIdx.x
                                  : (blockIdx.x & 1) * deal.half + set * (gridDim.x / 2) + (blockIdx.x >> 1);
  if (team >= deal.used) return;
  int64_t begin, end;
  diff_range(deal, team, begin, end);
  const int N = static_cast<int>(end - begin);
  if (N <= 0) return;

  auto uniform = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  auto enter = [&](DiffCursor& c) {   // the context fields of sequence c.b
    c.L = uniform(lens[c.b]);
    c.lo = diff_first(a, c.L);
    c.n = diff_stages(a, c.L);
  };
  auto place = [&](DiffCursor& c) {   // the fields of the worker's head block
    const int hb = (c.hg << a.team_shift) + member;
    c.pair = a.hb_per_pair == 1 ? hb : hb / a.hb_per_pair;
    c.head0 = c.pair * a.group + (hb - c.pair * a.hb_per_pair) * S::kHeads;
  };
  auto advance = [&](DiffCursor& c) {
    if (++c.st < c.n) return;
    c.st = 0;
    if (++c.hg == n_hg) {
      c.hg = 0;
      do ++c.b; while (c.b < a.batch - 1 && uniform(prefix[c.b + 1]) == uniform(prefix[c.b]));
      enter(c);
    }
    place(c);
  };
  DiffCursor cc;   // computing
  {
    int lo = 0, hi = a.batch - 1;   // the last sequence that begins at or before the range (its stages hold it)
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (static_cast<int64_t>(prefix[mid]) * n_hg <= begin) lo = mid;
      else hi = mid - 1;
    }
    cc.b = uniform(lo);
    enter(cc);
    const int rest = uniform(static_cast<int>(begin - static_cast<int64_t>(prefix[cc.b]) * n_hg));
    cc.hg = rest < cc.n ? 0 : rest / cc.n;
    cc.st = rest - cc.hg * cc.n;
    place(cc);
  }
  DiffCursor lc = cc, pc = cc;   // loading rows, loading page entries

  const u32 lds0 = uniform(static_cast<u32>(reinterpret_cast<uintptr_t>(smem)));
  const u32 ring_lds = lds0 + wave * S::kRing;
  const char* ring = smem + wave * S::kRing;
  const u32 page_lds = lds0 + S::kPageOff + wave * S::kPageSlots * 64;
  const int* page_mem = reinterpret_cast<const int*>(smem + S::kPageOff) + wave * S::kPageSlots * 16;
  const u32 query_lds = lds0 + S::kQueryOff + wave * S::kQueryBytes, lambda_lds = lds0 + S::kLambdaOff + wave * kWave * 4;
  const char* query_mem = smem + S::kQueryOff + wave * S::kQueryBytes;
  const float* lambda_mem = reinterpret_cast<const float*>(smem + S::kLambdaOff) + wave * kWave;

  // token (lane & 15) of a stage; what lies outside the attended range repeats its first or last token, so that every
  // row in LDS is one that the sequence owns (a probability of zero times a stale NaN would be NaN)
  auto token_of = [&](const DiffCursor& c) {
    const int t = (c.lo / kDiffTokens + c.st) * kDiffTokens + c16;
    return max(c.lo, min(t, c.L - 1));
  };
  auto split = [&](int t, int& col, int& off) {
    if (a.bs_shift >= 0) {
      col = t >> a.bs_shift;
      off = t & (a.block_size - 1);
    } else {
      col = static_cast<int>(static_cast<u32>(t) / static_cast<u32>(a.block_size));
      off = t - col * a.block_size;
    }
  };
  // Page entries of stage x (the cursor pc) into their slot.  Past the range the last stage's are fetched again: the
  // waits below count operations, and every stage has the same number of them.
  int px = 0;
  auto fetch_pages = [&]() {
    int col, off;
    split(token_of(pc), col, off);
    if (lane < 16) diff_dma4(a.block_table + pc.b * a.table_stride + col, page_lds + (px % S::kPageSlots) * 64);
    ++px;
    if (px < N) advance(pc);
  };
  // Row offsets of the next stage to load (the cursor lc), then its keys and its values.
  const int dc = lane % S::kChunks, dr = lane / S::kChunks;
  int lx = 0;
  int64_t row_off[NL];
  auto load_keys = [&]() {
    const int t = token_of(lc);
    int col, off;
    split(t, col, off);
    const int page = max(0, min(page_mem[(lx % S::kPageSlots) * 16 + c16], a.num_blocks - 1));
    const int slot = page * a.block_size + off;
    const u32 base = ring_lds + (lx % NS) * (2 * S::kTile);
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int row = i * S::kRowsPerLoad + dr;
      const int s = __shfl(slot, row, kWave);
      row_off[i] = s * a.row_bytes + lc.pair * S::kRow;
      diff_dma16(a.k_cache + row_off[i] + ((dc ^ row) & (S::kChunks - 1)) * 16, uniform(base + i * 1024));
    }
  };
  auto load_values = [&]() {
    const u32 base = ring_lds + (lx % NS) * (2 * S::kTile) + S::kTile;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int row = i * S::kRowsPerLoad + dr;
      diff_dma16(a.v_cache + row_off[i] + (dc ^ ((row & 7) << 1)) * 16, uniform(base + i * 1024));
    }
    ++lx;
    if (lx < N) advance(lc);
  };

  // Query rows [heads][2 maps][D] and lambdas of the context at cursor c.
  auto heads_of = [&](const DiffCursor& c) { return min(S::kHeads, (c.pair + 1) * a.group - c.head0); };
  auto fetch_query = [&](const DiffCursor& c) {
    const int heads = heads_of(c);
    const char* row = a.q + c.b * a.q_stride_bytes + static_cast<int64_t>(c.head0) * S::kRow;
#pragma unroll
    for (int i = 0; i < S::kQueryLoads; ++i)   // (what lies behind the block's heads repeats its last chunk)
      diff_dma16(row + min(i * kWave + lane, heads * S::kChunks - 1) * 16, uniform(query_lds + i * 1024));
    const int head = c.head0 + min(lane, heads - 1);
    diff_dma4(reinterpret_cast<const int32_t*>(a.lambda + c.b * a.lambda_batch_stride + head * a.lambda_head_stride),
              uniform(lambda_lds));
  };

  // ---- prologue: the first ring of stages in flight, the next ring's page entries with them
#pragma unroll 1
  for (int i = 0; i < NS; ++i) fetch_pages();
  fetch_query(cc);
  diff_wait_vm<0>();
#pragma unroll 1
  for (int i = 0; i < NS && i < N; ++i) {
    fetch_pages();
    load_keys();
    load_values();
  }

  // ---- the range
  u32x4 q[NB * KS];
  f32x4 o[NB][MB];
  float m[NB], l[NB];
  float lam = 0.0f;
  bool fresh = true;         // a context begins: its query rows are still to be read
  bool first_run = true;     // the first context of the range
  bool from_start = false;   // the context's first stage was this worker's
  const int k_read = c16 * S::kRow;
  const int v_row = 4 * g + (c16 >> 2);
  const int v_read = v_row * S::kRow + (c16 & 1) * 8;
  const int v_chunk = ((c16 & 3) >> 1) ^ ((v_row & 7) << 1);
  const int head = NB == 1 ? c16 & 7 : c16;   // the lane's head in its block

#pragma unroll 1
  for (int s = 0; s < N; ++s) {
    const int head0 = cc.head0, heads = heads_of(cc);
    const bool more = s + NS < N;
    const bool last = cc.st == cc.n - 1;
    DiffCursor nc = cc;
    if (s + 1 < N) advance(nc);
    const char* st = ring + (s % NS) * (2 * S::kTile);

    // ---- wait for the stage (and for the query rows of a new context, asked for one stage ago)
    if (s + NS > N) diff_wait_vm<0>();
    else if (NB == 1 && !(fresh && s > 0)) diff_wait_vm<(NS - 1) * kStageOps>();
    else if (fresh && s > 0) diff_wait_vm<kStageOps>();
    else diff_wait_vm<NL + (NS - 1) * kStageOps>();
    if (fresh) {
      fresh = false;
      from_start = cc.st == 0;
      lam = lambda_mem[head < heads ? head : 0];
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        if constexpr (S::kQueryLds) {   // (the lane's column belongs to map c16 / 8)
          q[kk] = *reinterpret_cast<const u32x4*>(query_mem + head * S::kRow + (c16 >> 3) * (2 * D) + g * 16 + kk * 64);
        } else {
          const char* row = a.q + cc.b * a.q_stride_bytes + static_cast<int64_t>(head0 + (head < heads ? head : 0)) * S::kRow +
                            g * 16 + kk * 64;
          // (columns without a head hold zeros; with the loads' registers used as they are the compiler moves them to
          // and from accumulation registers in the loop: 142 instead of 128 us for 64 sequences and 64 heads of 128 dims)
          const u32x4 x0 = ldg16(row), x1 = ldg16(row + 2 * D);
          q[kk] = head < heads ? x0 : u32x4{0, 0, 0, 0};
          q[(NB - 1) * KS + kk] = head < heads ? x1 : u32x4{0, 0, 0, 0};
        }
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        m[nb] = kNegBig;
        l[nb] = 0.0f;
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) o[nb][mb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
      diff_wait_lds();   // (the next context's rows may take the place of these)
    }
    if (last && s + 1 < N) fetch_query(nc);

    // ---- read the keys (and the values, where the registers hold both) and fill their place again
    u32x4 kr[2 * KS];
#pragma unroll
    for (int i = 0; i < 2 * KS; ++i)
      kr[i] = *reinterpret_cast<const u32x4*>(st + k_read + (((i * 4 + g) ^ c16) & (S::kChunks - 1)) * 16);
    constexpr int VB = MB / NB;
    s16x4 vt[VB];
    auto read_values = [&](int h) {
#pragma unroll
      for (int i = 0; i < VB; ++i)
        vt[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (diff_lds_s16x4*)(st + S::kTile + v_read + ((v_chunk ^ (2 * (h * VB + i))) * 16)));
      diff_wait_lds();
    };
    if constexpr (NB == 1) read_values(0);
    else diff_wait_lds();
    if (more) {
      fetch_pages();
      load_keys();
      if constexpr (NB == 1) load_values();
    }

    // ---- scores: lane (column c16, tokens 4 g .. 4 g + 3)
    f32x4 sc[NB];
    {
      f32x4 s0 = {0.0f, 0.0f, 0.0f, 0.0f}, s1 = s0;
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        s0 = Mfma<QT>::k32(kr[kk], q[kk], s0);
        s1 = Mfma<QT>::k32(kr[KS + kk], q[(NB - 1) * KS + kk], s1);
      }
      if constexpr (NB == 1) {
        // (both maps' keys met every column's queries: a column keeps its own map's scores)
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[0][r] = c16 < 8 ? s0[r] : s1[r];
      } else {
        sc[0] = s0;
        sc[NB - 1] = s1;
      }
    }
    const int tok0 = (cc.lo / kDiffTokens + cc.st) * kDiffTokens + 4 * g;
    u32x4 p[NB];   // the lane's four probabilities: their 16-bit values, then what those leave over
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float sv[4];
      bool over = false;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        sv[r] = tok0 + r < cc.L && tok0 + r >= cc.lo ? sc[nb][r] * a.scale_log2 : -INFINITY;
        over |= sv[r] - m[nb] > kTop;
      }
      if (__builtin_amdgcn_ballot_w64(over) != 0) {   // rare once the maxima have settled
        const float mx = diff_rows_max(fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3])));
        if (mx - m[nb] > kTop) {
          // (scores beyond 2^24, whose steps are wider than 1: where the lift is rounded up to 2^16 of weight, none)
          const float lifted = mx - DiffProbs<QT>::kLift, top = mx - lifted > kTop ? mx : lifted;
          const float alpha = fast_exp2(m[nb] - top);
          m[nb] = top;
          l[nb] *= alpha;
#pragma unroll
          for (int mb = 0; mb < MB; ++mb) o[nb][mb] *= alpha;
        }
      }
      float e[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        e[r] = fast_exp2(sv[r] - m[nb]);
        l[nb] += e[r];
      }
      const u32 h0 = QT::pack(e[0], e[1]), h1 = QT::pack(e[2], e[3]);
      p[nb] = u32x4{h0, h1, QT::pack(e[0] - QT::lo(h0), e[1] - QT::hi(h0)), QT::pack(e[2] - QT::lo(h1), e[3] - QT::hi(h1))};
    }

    // ---- values by the transposing read (lane c16 of 16 supplies 4 dims of token 4 g + c16 / 4 and receives the 4 tokens
    // 4 g .. of dim 16 mb + c16); two blocks of columns leave registers for half of them at a time
    if constexpr (NB == 2) {
      if (more) diff_wait_vm<(NS - 1) * kStageOps + 1 + NL>();
      else diff_wait_vm<0>();
    }
#pragma unroll
    for (int h = 0; h < NB; ++h) {
      if constexpr (NB == 2) {
        read_values(h);
        if (h == NB - 1 && more) load_values();
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < VB; ++i) {
          const int mb = h * VB + i;
          const u32x2 v = __builtin_bit_cast(u32x2, vt[i]);
          o[nb][mb] = Mfma<QT>::k32(u32x4{v[0], v[1], v[0], v[1]}, p[nb], o[nb][mb]);
        }
    }

    // ---- the end of the context, or of the range
    if (last || s == N - 1) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) l[nb] = diff_rows_sum(l[nb]);
      if (last && from_start) {
        const bool on = head < heads && (NB == 2 || c16 < 8);
        f32x4 d[MB];
        const float inv0 = 1.0f / l[0], inv1 = 1.0f / l[NB - 1];
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float v0 = o[0][mb][r] * inv0;
            // (one block: the same head's column of the other map is eight lanes on, row_ror:8)
            const float v1 = NB == 1 ? dpp<0x128>(v0) : o[NB - 1][mb][r] * inv1;
            d[mb][r] = diff_of(v0, lam, v1);
          }
        diff_store_row<QT, MB>(a, smem + S::kNormOff, d, cc.b, head0 + (head < heads ? head : 0), on, g);
      } else {
        const int64_t slot = 2 * ((static_cast<int64_t>(team) << a.team_shift) + member) + (first_run ? 0 : 1);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const int64_t col = slot * S::kCols + nb * 16 + c16;
          if (head < heads) {
            float* part = a.ws_o + col * (2 * D) + 4 * g;
            if (D == 128 && NB == 1 && a.stream_parts != 0) {
              int zero = 0;   // (an offset the compiler cannot see through: it folds the two branches' stores otherwise)
#pragma unroll
              for (int mb = 0; mb < MB; ++mb) {
                asm volatile("" : "+s"(zero));
                __builtin_nontemporal_store(o[nb][mb], reinterpret_cast<f32x4*>(part + zero + mb * 16));
              }
            } else {
#pragma unroll
              for (int mb = 0; mb < MB; ++mb) *reinterpret_cast<f32x4*>(part + mb * 16) = o[nb][mb];
            }
            if (g == 0) *reinterpret_cast<f32x2*>(a.ws_ml + col * 2) = f32x2{m[nb], l[nb]};
          }
        }
      }
      first_run = false;
      fresh = true;
    }
    cc = nc;
  }
}

// Joins the parts of the contexts that several teams hold, and writes zeros for empty contexts.  A lane holds 2 D / 64 dims
// of both maps.  SPLIT: one workgroup per (head, sequence), whose WAVES wavefronts share the parts; else one wavefront per
// head, WAVES heads to a workgroup.  The parts are added in an order that only their number sets.
template <typename QT, int D, int NB, int WAVES, bool SPLIT>
__global__ __launch_bounds__(WAVES * kWave) void diff_merge_kernel(DiffArgs a) {
  using S = DiffShape<D, NB>;
  constexpr int E = 2 * D / kWave;   // dims per lane
  typedef __attribute__((ext_vector_type(E))) float fvec;
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = SPLIT ? blockIdx.x : blockIdx.x * WAVES + wave, b = blockIdx.y;
  if (!SPLIT && head >= a.n_heads) return;
  const int pair = a.group == 1 ? head : static_cast<int>(static_cast<u32>(head) / static_cast<u32>(a.group));
  const int in_pair = head - pair * a.group;
  const int hb = pair * a.hb_per_pair + static_cast<int>(static_cast<u32>(in_pair) / S::kHeads);
  const int h = static_cast<int>(static_cast<u32>(in_pair) % S::kHeads);
  const int n_hg = (a.n_pairs * a.hb_per_pair) >> a.team_shift;
  const int hg = hb >> a.team_shift, member = hb & ((1 << a.team_shift) - 1);
  // (asked for before the parts, whose loads hang off the prefix: the launch is a chain of such trips)
  const float lam = a.lambda[b * a.lambda_batch_stride + head * a.lambda_head_stride];
  u32 weight[E / 2];
#pragma unroll
  for (int i = 0; i < E / 2; ++i) weight[i] = a.norm_w != nullptr ? reinterpret_cast<const u32*>(a.norm_w)[lane * (E / 2) + i] : 0;
  const int p0 = a.ws_prefix[b], n = a.ws_prefix[b + 1] - p0;
  char* row = a.out + b * a.out_stride_bytes + static_cast<int64_t>(head) * (4 * D);
  if (n == 0) {
    if (!SPLIT || wave == 0)
      for (int i = 0; i < E / 2; ++i) reinterpret_cast<u32*>(row)[lane * (E / 2) + i] = 0;
    return;
  }
  const DiffDeal deal = diff_deal(a, static_cast<int64_t>(a.ws_prefix[a.batch]) * n_hg);
  const int64_t s0 = static_cast<int64_t>(p0) * n_hg + static_cast<int64_t>(hg) * n;
  int64_t begin, unused;
  const int wf = diff_team_of(deal, s0, begin), wl = diff_team_of(deal, s0 + n - 1, unused);
  if (wf == wl) return;   // one team held it whole and wrote the rows
  const int first_slot = begin < s0 ? 1 : 0;
  fvec o[2];
  float m[2], l[2];
#pragma unroll
  for (int mp = 0; mp < 2; ++mp) {
    o[mp] = fvec(0.0f);
    m[mp] = kNegBig;
    l[mp] = 0.0f;
  }
#pragma unroll 4
  for (int w = wf + (SPLIT ? wave : 0); w <= wl; w += SPLIT ? WAVES : 1) {
    const int64_t slot = 2 * ((static_cast<int64_t>(w) << a.team_shift) + member) + (w == wf ? first_slot : 0);
#pragma unroll
    for (int mp = 0; mp < 2; ++mp) {
      const int64_t col = slot * S::kCols + (NB == 1 ? mp * 8 : mp * 16) + h;
      const f32x2 ml = *reinterpret_cast<const f32x2*>(a.ws_ml + col * 2);
      const fvec x = *reinterpret_cast<const fvec*>(a.ws_o + col * (2 * D) + lane * E);
      const float mx = fmaxf(m[mp], ml[0]);
      const float f0 = fast_exp2(m[mp] - mx), f1 = fast_exp2(ml[0] - mx);
      o[mp] = o[mp] * f0 + x * f1;
      l[mp] = l[mp] * f0 + ml[1] * f1;
      m[mp] = mx;
    }
  }
  if constexpr (SPLIT) {
    __shared__ float acc[WAVES][2][2 * D];
    __shared__ float sums[WAVES][2][2];   // maximum, sum
#pragma unroll
    for (int mp = 0; mp < 2; ++mp) {
      *reinterpret_cast<fvec*>(&acc[wave][mp][lane * E]) = o[mp];
      if (lane == 0) {
        sums[wave][mp][0] = m[mp];
        sums[wave][mp][1] = l[mp];
      }
    }
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int mp = 0; mp < 2; ++mp) {
      float mx = m[mp];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) mx = fmaxf(mx, sums[w][mp][0]);
      fvec t = fvec(0.0f);
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const float f = fast_exp2(sums[w][mp][0] - mx);
        t += *reinterpret_cast<const fvec*>(&acc[w][mp][lane * E]) * f;
        sum += sums[w][mp][1] * f;
      }
      o[mp] = t;
      l[mp] = sum;
    }
  }
#pragma unroll
  for (int mp = 0; mp < 2; ++mp) o[mp] *= 1.0f / l[mp];
  fvec d;
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < E; ++i) d[i] = diff_of(o[0][i], lam, o[1][i]);
#pragma unroll
  for (int i = 0; i < E; ++i) ss += d[i] * d[i];
  ss = group_sum<32>(ss);
  ss += __shfl_xor(ss, 32, kWave);
  float f = a.out_scale;
  if (a.norm_w != nullptr) f *= 1.0f / __builtin_sqrtf(ss / static_cast<float>(2 * D) + a.eps);
#pragma unroll
  for (int i = 0; i < E; i += 2) {
    float w0 = 1.0f, w1 = 1.0f;
    if (a.norm_w != nullptr) {
      w0 = QT::lo(weight[i / 2]);
      w1 = QT::hi(weight[i / 2]);
    }
    reinterpret_cast<u32*>(row)[(lane * E + i) / 2] = QT::pack(d[i] * f * w0, d[i + 1] * f * w1);
  }
}

template <typename QT, int D, int NB>
int launch_diff(const DiffArgs& a, hipStream_t stream) {
  using S = DiffShape<D, NB>;
  static std::atomic<uint64_t> configured{0};
  const hipError_t e = once_per_device(configured, [] {
    return hipFuncSetAttribute(reinterpret_cast<const void*>(diff_decode_kernel<QT, D, NB>),
                               hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(S::lds_bytes(kDiffMaxBatch)));
  });
  if (e != hipSuccess) return static_cast<int>(e);
  launch_timed(diff_decode_kernel<QT, D, NB>, dim3(static_cast<unsigned>(a.n_workers / S::kWaves)), dim3(S::kThreads),
               S::lds_bytes(a.batch), stream, a);
  int rc = static_cast<int>(hipGetLastError());
  if (rc != 0) return rc;
  // few rows: their contexts may be in many parts, which the wavefronts of a workgroup share; many rows: a wavefront each
  const unsigned batch = static_cast<unsigned>(a.batch), heads = static_cast<unsigned>(a.n_heads);
  const int64_t rows = static_cast<int64_t>(a.batch) * a.n_heads;
  // (parts of a row: the teams by the contexts that share them, or what the table or the window leaves to split)
  const int64_t shared = (a.n_workers >> a.team_shift) / (static_cast<int64_t>(a.batch) * ((a.n_pairs * a.hb_per_pair) >> a.team_shift));
  const int64_t stages = (a.window_left >= 0 && a.window_left < a.max_len ? a.window_left : a.max_len) / kDiffTokens;
  if (rows <= kDiffSplit8 && shared > kDiffManyParts && stages > kDiffManyParts)
    launch_timed(diff_merge_kernel<QT, D, NB, 16, true>, dim3(heads, batch), dim3(16 * kWave), 0, stream, a);
  else if (rows <= kDiffSplit8)
    launch_timed(diff_merge_kernel<QT, D, NB, 8, true>, dim3(heads, batch), dim3(8 * kWave), 0, stream, a);
  else if (rows <= kDiffSplit4)
    launch_timed(diff_merge_kernel<QT, D, NB, 4, true>, dim3(heads, batch), dim3(4 * kWave), 0, stream, a);
  else
    launch_timed(diff_merge_kernel<QT, D, NB, 4, false>, dim3((heads + 3) / 4, batch), dim3(4 * kWave), 0, stream, a);
  return static_cast<int>(hipGetLastError());
}

template <typename QT>
int dispatch_diff(const DiffArgs& a, int64_t head_dim, hipStream_t stream) {
  if (head_dim == 64) return a.group <= 8 ? launch_diff<QT, 64, 1>(a, stream) : launch_diff<QT, 64, 2>(a, stream);
  return a.group <= 8 ? launch_diff<QT, 128, 1>(a, stream) : launch_diff<QT, 128, 2>(a, stream);
}

size_t diff_prefix_bytes() { return (static_cast<size_t>(kDiffMaxBatch + 1) * 4 + 255) / 256 * 256; }
int64_t diff_columns(int64_t group) { return group <= 8 ? 16 : 32; }
int64_t diff_workers(int64_t head_dim, int64_t group) {
  const int waves = head_dim == 64 ? (group <= 8 ? DiffShape<64, 1>::kWaves : DiffShape<64, 2>::kWaves)
                                   : (group <= 8 ? DiffShape<128, 1>::kWaves : DiffShape<128, 2>::kWaves);
  return static_cast<int64_t>(device_cu_count()) * waves;
}

}  // namespace

// prefix | maxima and sums | partial rows, two slots per worker
size_t diff_workspace_bytes(int64_t n_heads, int64_t n_pairs, int64_t head_dim) {
  if (n_heads <= 0 || n_pairs <= 0 || n_heads % n_pairs != 0 || (head_dim != 64 && head_dim != 128)) return 0;
  const size_t cols = static_cast<size_t>(diff_workers(head_dim, n_heads / n_pairs) * 2 * diff_columns(n_heads / n_pairs));
  return diff_prefix_bytes() + cols * 2 * 4 + cols * 2 * head_dim * 4;
}

int paged_decode_diff(const void* q, const void* k_cache, const void* v_cache, void* out, const int32_t* block_table,
                      int64_t table_stride, int64_t table_width, const int32_t* seq_lens, const float* lambda,
                      int64_t lambda_batch_stride, int64_t lambda_head_stride, const void* norm_weight, float eps,
                      float out_scale, int64_t batch, int64_t n_heads, int64_t n_kv_pairs, int64_t head_dim,
                      int64_t block_size, int64_t num_blocks, int64_t q_token_stride, int64_t out_token_stride,
                      int64_t window_left, float sm_scale, void* workspace, size_t workspace_bytes, int dtype,
                      hipStream_t stream) {
  if (batch == 0) return XLLM_MI355_OK;
  if (q == nullptr || k_cache == nullptr || v_cache == nullptr || out == nullptr || block_table == nullptr ||
      seq_lens == nullptr || lambda == nullptr)
    return XLLM_MI355_EINVAL;
  if (batch < 0 || n_heads <= 0 || n_kv_pairs <= 0 || n_heads % n_kv_pairs != 0 || n_heads > 65535 || block_size <= 0 ||
      num_blocks <= 0 || table_width <= 0 || table_stride < table_width || !(sm_scale > 0.0f) || !(eps >= 0.0f) ||
      lambda_batch_stride < 0 || lambda_head_stride < 0)
    return XLLM_MI355_EINVAL;
  if (dtype != XLLM_MI355_BF16 && dtype != XLLM_MI355_FP16) return XLLM_MI355_EDTYPE;
  if (head_dim != 64 && head_dim != 128) return XLLM_MI355_ESHAPE;
  if (block_size > 0x7fffffffLL || num_blocks > 0x7fffffffLL || num_blocks * block_size > 0x7fffffffLL)
    return XLLM_MI355_ESHAPE;
  if (q_token_stride < 2 * n_heads * head_dim || out_token_stride < 2 * n_heads * head_dim) return XLLM_MI355_EINVAL;
  auto aligned = [](const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  if (!aligned(q, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16) || (q_token_stride & 7) != 0 || !aligned(out, 8) ||
      (out_token_stride & 3) != 0 || !aligned(norm_weight, 8))
    return XLLM_MI355_EALIGN;
  const int64_t group = n_heads / n_kv_pairs, hb_per_pair = group <= 8 ? 1 : (group + 15) / 16;
  const int64_t head_blocks = n_kv_pairs * hb_per_pair;
  const int team_shift = head_blocks % 4 == 0 ? 2 : head_blocks % 2 == 0 ? 1 : 0;
  const int64_t max_len = table_width > (0x7fffffffLL - 16) / block_size ? 0x7fffffffLL - 16 : table_width * block_size;
  const int64_t attended = window_left >= 0 && window_left < max_len ? window_left + 1 : max_len;
  // stages of one sequence, at most (attended tokens that do not begin at a stage reach into one more)
  const int64_t most_stages = (attended / kDiffTokens + 2) * (head_blocks >> team_shift);
  if (most_stages > 0x7fffffffLL) return XLLM_MI355_ESHAPE;
  const size_t need = diff_workspace_bytes(n_heads, n_kv_pairs, head_dim);
  if (workspace == nullptr || !aligned(workspace, 256) || workspace_bytes < need) return XLLM_MI355_EWORKSPACE;

  {
    const int64_t cache = num_blocks * block_size * n_kv_pairs * head_dim * 4, row = 2 * n_heads * head_dim;
    const Span out_rows = span_of(out, batch, out_token_stride, 1, 0, row, 2), space(workspace, static_cast<int64_t>(need));
    for (const Span& r : {span_of(q, batch, q_token_stride, 1, 0, row, 2), Span(k_cache, cache), Span(v_cache, cache),
                          span_of(block_table, batch, table_stride, 1, 0, table_width, 4), Span(seq_lens, batch * 4),
                          span_of(lambda, batch, lambda_batch_stride, n_heads, lambda_head_stride, 1, 4),
                          Span(norm_weight, norm_weight != nullptr ? 4 * head_dim : 0)})
      if (out_rows.meets(r) || space.meets(r)) return XLLM_MI355_EINVAL;
    if (out_rows.meets(space)) return XLLM_MI355_EINVAL;
  }
  DiffArgs a = {};
  a.n_heads = static_cast<int>(n_heads);
  a.n_pairs = static_cast<int>(n_kv_pairs);
  a.group = static_cast<int>(group);
  a.hb_per_pair = static_cast<int>(hb_per_pair);
  a.block_size = static_cast<int>(block_size);
  a.bs_shift = -1;
  for (int s = 0; s < 31; ++s)
    if ((1LL << s) == block_size) a.bs_shift = s;
  a.num_blocks = static_cast<int>(num_blocks);
  a.max_len = static_cast<int>(max_len);
  a.window_left = window_left < 0 ? -1 : static_cast<int>(window_left < 0x7fffffffLL ? window_left : 0x7fffffffLL);
  a.n_workers = static_cast<int>(diff_workers(head_dim, a.group));
  a.pools = device_cu_count() == 256 ? 1 : 0;
  a.team_shift = team_shift;
  a.scale_log2 = sm_scale * kLog2e;
  a.eps = eps;
  a.out_scale = out_scale;
  a.k_cache = static_cast<const char*>(k_cache);
  a.v_cache = static_cast<const char*>(v_cache);
  a.norm_w = static_cast<const char*>(norm_weight);
  a.table_stride = table_stride;
  a.q_stride_bytes = q_token_stride * 2;
  a.out_stride_bytes = out_token_stride * 2;
  a.row_bytes = n_kv_pairs * head_dim * 4;
  a.lambda_batch_stride = lambda_batch_stride;
  a.lambda_head_stride = lambda_head_stride;
  char* ws = static_cast<char*>(workspace);
  const size_t cols = static_cast<size_t>(a.n_workers) * 2 * diff_columns(a.group);
  a.ws_prefix = reinterpret_cast<int*>(ws);
  a.ws_ml = reinterpret_cast<float*>(ws + diff_prefix_bytes());
  a.ws_o = a.ws_ml + cols * 2;
  // batches beyond the LDS prefix, or whose tables could hold more stages than 32 bits count, are decoded in slices, one
  // launch pair after the other
  const int64_t fit = 0x7fffffffLL / most_stages, slice = fit < kDiffMaxBatch ? fit : kDiffMaxBatch;
  for (int64_t b0 = 0; b0 < batch; b0 += slice) {
    a.batch = static_cast<int>(batch - b0 < slice ? batch - b0 : slice);
    a.q = static_cast<const char*>(q) + b0 * a.q_stride_bytes;
    a.out = static_cast<char*>(out) + b0 * a.out_stride_bytes;
    a.block_table = block_table + b0 * table_stride;
    a.seq_lens = seq_lens + b0;
    a.lambda = lambda + b0 * lambda_batch_stride;
    a.stream_parts = a.batch * n_heads >= kDiffStreamRows ? 1 : 0;
    const int rc = dtype == XLLM_MI355_BF16 ? dispatch_diff<BF16>(a, head_dim, stream) : dispatch_diff<FP16>(a, head_dim, stream);
    if (rc != 0) return rc;
  }
  return XLLM_MI355_OK;
}

}  // namespace xllm_mi355
