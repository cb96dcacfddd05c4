// Rotary positions outside the fused qkv buffer (rope_and_cache.hip serves that one), for gfx950:
//   rope_cos_sin             cos | sin rows of positions, from frequencies that may be scaled for long contexts
//   rotary_embedding         rotation of q and k held in tensors of their own, part of the head, either pair layout, and
//                            its transpose (the inverse rotation, which is also its gradient)
//   mla_norm_rope_and_cache  the MLA counterpart of rope_and_cache: RMS norm of the latent, rotation of the rope keys and
//                            queries, and the store into the latent cache
//
// Pairs are (a, b) = (x[2i], x[2i+1]) when interleaved, (x[i], x[i + R/2]) otherwise:
//   (a, b) -> (a c_i - b s_i, b c_i + a s_i)
// in fp32 between one load and one store.  All three are bound by the bytes they move (a few operations per element) or,
// at decode sizes, by the launch: the kernels read and write 16 bytes per lane and instruction and keep several in flight.
// 64 rows of 128 values take 2.2 us, the rotation of 64 tokens of 40 heads and the MLA prologue of 64 tokens of 128 heads
// 3.0 us each, which is a launch with one or two trips to memory in it (position, then its cos | sin row).
#include "common.cuh"
#include "launch.h"

namespace xllm_mi355 {

namespace {

constexpr int kRotThreads = 256;
constexpr int64_t kRotGroups = 0xffffffffLL / kRotThreads;   // a launch counts its threads in 32 bits

// ---- element types ------------------------------------------------------------------------------------------------

template <int DT>
struct Elem;
template <>
struct Elem<XLLM_MI355_BF16> {
  using T = uint16_t;
  static __device__ __forceinline__ float get(T x) { return BF16::to_f32(x); }
  static __device__ __forceinline__ T put(float x) { return BF16::from_f32(x); }
};
template <>
struct Elem<XLLM_MI355_FP16> {
  using T = uint16_t;
  static __device__ __forceinline__ float get(T x) { return FP16::to_f32(x); }
  static __device__ __forceinline__ T put(float x) { return FP16::from_f32(x); }
};
template <>
struct Elem<XLLM_MI355_FP32> {
  using T = float;
  static __device__ __forceinline__ float get(T x) { return x; }
  static __device__ __forceinline__ T put(float x) { return x; }
};

// N elements as 16-byte words.
template <int DT, int N>
struct Pack {
  using T = typename Elem<DT>::T;
  static constexpr int kWords = N * static_cast<int>(sizeof(T)) / 16;
  static_assert(kWords >= 1 && kWords * 16 == N * static_cast<int>(sizeof(T)), "whole 16-byte words");
  u32x4 w[kWords];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = reinterpret_cast<const u32x4*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) reinterpret_cast<u32x4*>(p)[i] = w[i];
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (DT == XLLM_MI355_FP32) {
      return as_f32(w[i / 4][i % 4]);
    } else {
      const u32 x = w[i / 8][(i / 2) % 4];
      return Elem<DT>::get(static_cast<uint16_t>((i & 1) ? x >> 16 : x & 0xffffu));
    }
  }
  // elements 2 i and 2 i + 1
  __device__ __forceinline__ void put2(int i, float a, float b) {
    if constexpr (DT == XLLM_MI355_FP32) {
      w[i / 2][(2 * i) % 4] = as_u32(a);
      w[i / 2][(2 * i) % 4 + 1] = as_u32(b);
    } else if constexpr (DT == XLLM_MI355_BF16) {
      w[i / 4][i % 4] = BF16::pack(a, b);
    } else {
      w[i / 4][i % 4] = FP16::pack(a, b);
    }
  }
};

// ---- cos | sin rows ------------------------------------------------------------------------------------------------

// cos and sin of `angle` in 64 bits: the multiple q of pi / 2 is taken off in two parts (its product with the leading part is
// exact inside the fused multiply-add, so what is left of angles up to 2^50 is good to 2^-52 of the angle), then polynomials
// in r^2 on [-pi/4, pi/4], fitted for the smallest largest error of sin r (2.4e-12) and cos r (5.4e-11, a thousandth of an
// fp32 step) with their leading terms r and 1 kept, so that position 0 gives 1 and 0.  Adding 1.5 2^52 rounds to an integer
// and leaves it in the low bits of the sum: conversions and roundings in 64 bits run at a fraction of the rate of products.
struct Quarter {   // sin and cos of what is left, and q mod 4
  double s, c;
  u32 k;
};
__device__ __forceinline__ Quarter sin_cos_64(double angle) {
  constexpr double kShift = 6755399441055744.0;
  const double shifted = __builtin_fma(angle, 0.63661977236758134308, kShift);
  const double q = shifted - kShift;
  double r = __builtin_fma(-q, 1.5707963267948965580, angle);
  r = __builtin_fma(-q, 6.1232339957367660359e-17, r);
  const double z = r * r;
  double ps = 2.716013937443816e-06, pc = 2.4390449888022627e-05;
  ps = __builtin_fma(ps, z, -0.0001983904376152292);
  ps = __builtin_fma(ps, z, 0.00833332823868483);
  ps = __builtin_fma(ps, z, -0.16666666627998758);
  pc = __builtin_fma(pc, z, -0.0013886763785924106);
  pc = __builtin_fma(pc, z, 0.041666623324085626);
  pc = __builtin_fma(pc, z, -0.4999999972510603);
  return {__builtin_fma(r * z, ps, r), __builtin_fma(pc, z, 1.0), static_cast<u32>(__builtin_bit_cast(uint64_t, shifted))};
}

// V pairs of the row of a position, times `factor`, rounded to fp32 (and from there to the 16-bit types).  Quadrant and signs
// are settled on the rounded results: comparisons in 64 bits were a fifth of the operations.
template <int V>
__device__ __forceinline__ void row_pairs(double pos, const double (&freq)[V], double factor, float (&c)[V], float (&s)[V]) {
  Quarter t[V];
#pragma unroll
  for (int i = 0; i < V; ++i) t[i] = sin_cos_64(pos * freq[i]);
  if (factor != 1.0) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      t[i].s *= factor;
      t[i].c *= factor;
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float sr = static_cast<float>(t[i].s), cr = static_cast<float>(t[i].c);
    const bool swap = (t[i].k & 1u) != 0;
    c[i] = as_f32(as_u32(swap ? sr : cr) ^ ((t[i].k + 1u) & 2u) << 30);
    s[i] = as_f32(as_u32(swap ? cr : sr) ^ (t[i].k & 2u) << 30);
  }
}

// Every row is made by the formula above from its own position, so that a position has the same bits in a table made at load,
// in a range of any length and in a step's listed rows.  (Turning a row into the next ones by its frequencies, one evaluation
// for eight, took 12.8 us for 131072 rows of 128 fp32 values and 9.4 us of bf16; but a turned angle is not the rounded product
// that a listed position has, and some values fell on the other side of their rounding.)
// One lane makes V consecutive pairs of a row: V cosines and V sines, 16 bytes of each where the row allows it.  Bound by the
// launch (64 rows of 128 values: 2.1 us), beyond that by 17 operations in 64 bits a pair, at half the rate of those in 32, on
// top of the stores: 131072 rows of 128 values 14.0 us in fp32, where the stores alone take 11.9 us and a plain fill of as many
// bytes 11.4 us, and 13.3 us in bf16.  (Several rows a lane: the same.)
template <int DT, int V>
__global__ __launch_bounds__(kRotThreads) void rope_cos_sin_kernel(const double* inv_freq, const int64_t* positions,
                                                                   int64_t first, int64_t n_units, int half, double factor,
                                                                   typename Elem<DT>::T* out) {
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kRotThreads + threadIdx.x;
  if (unit >= n_units) return;
  const int per = half / V;
  // (32-bit division where it fits, which is every table below 2^31 lanes)
  const int64_t row = n_units <= 0x7fffffffLL ? static_cast<u32>(unit) / static_cast<u32>(per) : unit / per;
  const int i0 = static_cast<int>(unit - row * per) * V;
  const double pos = static_cast<double>(positions != nullptr ? positions[row] : first + row);
  double freq[V];
#pragma unroll
  for (int i = 0; i < V; ++i) freq[i] = inv_freq[i0 + i];
  typename Elem<DT>::T* p = out + row * (2 * static_cast<int64_t>(half)) + i0;
  float c[V], s[V];
  row_pairs<V>(pos, freq, factor, c, s);
  if constexpr (V == 1) {
    p[0] = Elem<DT>::put(c[0]);
    p[half] = Elem<DT>::put(s[0]);
  } else {
    Pack<DT, V> a, b;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      a.put2(i, c[2 * i], c[2 * i + 1]);
      b.put2(i, s[2 * i], s[2 * i + 1]);
    }
    a.store(p);
    b.store(p + half);
  }
}

template <int DT>
int launch_cos_sin(const double* inv_freq, const int64_t* positions, int64_t first, int64_t rows, int64_t half,
                   double factor, void* out, hipStream_t stream) {
  constexpr int V = DT == XLLM_MI355_FP32 ? 4 : 8;
  using T = typename Elem<DT>::T;
  const bool wide = half % V == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  const int64_t units = rows * (wide ? half / V : half);
  const int64_t groups = (units + kRotThreads - 1) / kRotThreads;
  if (groups > kRotGroups) return XLLM_MI355_ESHAPE;
  const dim3 grid(static_cast<unsigned>(groups));
  if (wide)
    rope_cos_sin_kernel<DT, V><<<grid, kRotThreads, 0, stream>>>(inv_freq, positions, first, units, static_cast<int>(half),
                                                                 factor, static_cast<T*>(out));
  else
    rope_cos_sin_kernel<DT, 1><<<grid, kRotThreads, 0, stream>>>(inv_freq, positions, first, units, static_cast<int>(half),
                                                                 factor, static_cast<T*>(out));
  return static_cast<int>(hipGetLastError());
}

// ---- rotation ------------------------------------------------------------------------------------------------------

struct RotSide {            // q or k; strides in elements
  const char* in;
  char* out;
  int64_t in_token, in_head, out_token, out_head;
  int heads, dim, offset;
};

struct RotArgs {
  RotSide q, k;
  const int64_t* positions;
  const char* cos_sin;
  int64_t n_positions;      // rows of cos_sin; a position outside [0, n_positions) is not rotated
  int64_t n_units;
  int rot;                  // rotated dims R
  int rot_units;            // lanes per head and rotated part
  int units;                // lanes per head: the rotated part, and for out of place the rest of the wider side
};

// cos and sin of pairs [i, i + P) of a table row.
template <int CT, int P, bool VEC>
__device__ __forceinline__ void rot_row(const char* table, int64_t row, int rot, int i, float (&c)[P], float (&s)[P]) {
  using T = typename Elem<CT>::T;
  const T* p = reinterpret_cast<const T*>(table) + row * rot + i;
  if constexpr (VEC && P * sizeof(T) >= 16) {
    Pack<CT, P> a, b;
    a.load(p);
    b.load(p + rot / 2);
#pragma unroll
    for (int j = 0; j < P; ++j) {
      c[j] = a.get(j);
      s[j] = b.get(j);
    }
  } else {
#pragma unroll
    for (int j = 0; j < P; ++j) {
      c[j] = Elem<CT>::get(p[j]);
      s[j] = Elem<CT>::get(p[rot / 2 + j]);
    }
  }
}

// P pairs in two 16-byte words: their first and second elements, or P / 2 pairs in each word when interleaved.
template <int DT, int P, bool INTERLEAVE>
__device__ __forceinline__ void turn_words(Pack<DT, P>& x, Pack<DT, P>& y, const float (&c)[P], const float (&s)[P]) {
  if constexpr (INTERLEAVE) {
#pragma unroll
    for (int j = 0; j < P; ++j) {
      Pack<DT, P>& w = j < P / 2 ? x : y;
      const int e = j < P / 2 ? j : j - P / 2;
      const float p0 = w.get(2 * e), p1 = w.get(2 * e + 1);
      w.put2(e, __builtin_fmaf(p0, c[j], -(p1 * s[j])), __builtin_fmaf(p1, c[j], p0 * s[j]));
    }
  } else {
#pragma unroll
    for (int j = 0; j < P; j += 2) {
      const float a0 = x.get(j), a1 = x.get(j + 1), b0 = y.get(j), b1 = y.get(j + 1);
      x.put2(j / 2, __builtin_fmaf(a0, c[j], -(b0 * s[j])), __builtin_fmaf(a1, c[j + 1], -(b1 * s[j + 1])));
      y.put2(j / 2, __builtin_fmaf(b0, c[j], a0 * s[j]), __builtin_fmaf(b1, c[j + 1], a1 * s[j + 1]));
    }
  }
}

// A lane owns P pairs of a head (P = 16 bytes of elements, so two 16-byte words: the pairs' two halves, or two neighbouring
// words when interleaved).  Lanes behind the rotated part copy the rest of the head when the result goes elsewhere, two
// words each, at neighbouring words in neighbouring lanes.  One head per lane: with four (one set of cosines and sines for
// all of them, four times the bytes in flight per lane) 8192 tokens of 40 heads took the same 27 us, 4097 tokens of 20
// heads with a copied rest 28 instead of 19 us, for want of wavefronts.  Bound by the bytes: 8192 tokens of 40 heads of 128
// bf16 values (172 MB with the table's rows) 27.2 us to another place = 6.3 TB/s and 27.9 us in place, 4097 tokens of 20 heads of 256 fp16 values to
// another place, 64 of them rotated (84 MB), 17.2 us = 4.9 TB/s; a large copy runs at 5.2 TB/s.
// VEC = false takes one pair (or two elements to copy) per lane, for operands that are not aligned to 16 bytes.
template <int DT, int CT, bool INTERLEAVE, bool VEC>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(RotArgs a, float sin_sign) {
  using T = typename Elem<DT>::T;
  constexpr int P = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * kRotThreads + threadIdx.x;
  if (idx >= a.n_units) return;
  const int heads = a.q.heads + a.k.heads;
  int64_t token;
  int unit, head;
  if (a.n_units <= 0x7fffffffLL) {
    const u32 r = static_cast<u32>(idx) / static_cast<u32>(a.units);
    unit = static_cast<int>(static_cast<u32>(idx) - r * static_cast<u32>(a.units));
    const u32 t = r / static_cast<u32>(heads);
    head = static_cast<int>(r - t * static_cast<u32>(heads));
    token = t;
  } else {
    const int64_t r = idx / a.units;
    unit = static_cast<int>(idx - r * a.units);
    token = r / heads;
    head = static_cast<int>(r - token * heads);
  }
  const bool is_q = head < a.q.heads;
  const RotSide& sd = is_q ? a.q : a.k;
  if (!is_q) head -= a.q.heads;
  const T* in = reinterpret_cast<const T*>(sd.in) + token * sd.in_token + head * sd.in_head;
  T* out = reinterpret_cast<T*>(sd.out) + token * sd.out_token + head * sd.out_head;

  if (unit >= a.rot_units) {   // the rest of the head: what lies before the rotated part, then what lies behind it
    if (sd.in == sd.out) return;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const int e = (unit - a.rot_units + w * (a.units - a.rot_units)) * P;
      if (e >= sd.dim - a.rot) break;
      const int d = e < sd.offset ? e : e + a.rot;
      if constexpr (VEC) {
        Pack<DT, P> x;
        x.load(in + d);
        x.store(out + d);
      } else {
        out[d] = in[d];
      }
    }
    return;
  }

  const int i = unit * P;                                                    // first pair
  const int da = sd.offset + (INTERLEAVE ? 2 * i : i);                       // where the pairs' words lie
  const int db = sd.offset + (INTERLEAVE ? 2 * i + P : i + a.rot / 2);
  const int64_t pos = a.positions[token];
  const bool turn = pos >= 0 && pos < a.n_positions;
  if constexpr (VEC) {
    Pack<DT, P> x, y;
    x.load(in + da);
    y.load(in + db);
    if (turn) {
      float c[P], s[P];
      rot_row<CT, P, true>(a.cos_sin, pos, a.rot, i, c, s);
#pragma unroll
      for (int j = 0; j < P; ++j) s[j] *= sin_sign;
      turn_words<DT, P, INTERLEAVE>(x, y, c, s);
    }
    x.store(out + da);
    y.store(out + db);
  } else {
    const T xa = in[da], xb = in[db];
    float c[1] = {1.0f}, s[1] = {0.0f};
    if (turn) rot_row<CT, 1, false>(a.cos_sin, pos, a.rot, i, c, s);
    s[0] *= sin_sign;
    const float p0 = Elem<DT>::get(xa), p1 = Elem<DT>::get(xb);
    out[da] = turn ? Elem<DT>::put(__builtin_fmaf(p0, c[0], -(p1 * s[0]))) : xa;
    out[db] = turn ? Elem<DT>::put(__builtin_fmaf(p1, c[0], p0 * s[0])) : xb;
  }
}

template <int DT, int CT, bool INTERLEAVE, bool VEC>
int launch_rotary(RotArgs a, bool copy_rest, int inverse, int64_t n_tokens, hipStream_t stream) {
  constexpr int P = VEC ? 16 / static_cast<int>(sizeof(typename Elem<DT>::T)) : 1;
  a.rot_units = a.rot / 2 / P;
  const int wide = a.k.heads > 0 && a.k.dim > a.q.dim ? a.k.dim : a.q.dim;
  a.units = a.rot_units + (copy_rest ? (wide - a.rot + 2 * P - 1) / (2 * P) : 0);
  a.n_units = n_tokens * (a.q.heads + a.k.heads) * a.units;
  const int64_t groups = (a.n_units + kRotThreads - 1) / kRotThreads;
  if (groups > kRotGroups) return XLLM_MI355_ESHAPE;
  rotary_kernel<DT, CT, INTERLEAVE, VEC><<<dim3(static_cast<unsigned>(groups)), kRotThreads, 0, stream>>>(
      a, inverse != 0 ? -1.0f : 1.0f);
  return static_cast<int>(hipGetLastError());
}

template <int DT>
int dispatch_rotary(const RotArgs& a, int cos_sin_dtype, int interleave, bool vec, bool copy_rest, int inverse,
                    int64_t n_tokens, hipStream_t stream) {
#define XLLM_ROT(CT)                                                                                            \
  (interleave != 0 ? (vec ? launch_rotary<DT, CT, true, true>(a, copy_rest, inverse, n_tokens, stream)          \
                          : launch_rotary<DT, CT, true, false>(a, copy_rest, inverse, n_tokens, stream))        \
                   : (vec ? launch_rotary<DT, CT, false, true>(a, copy_rest, inverse, n_tokens, stream)         \
                          : launch_rotary<DT, CT, false, false>(a, copy_rest, inverse, n_tokens, stream)))
  switch (cos_sin_dtype) {
    case XLLM_MI355_FP32: return XLLM_ROT(XLLM_MI355_FP32);
    case XLLM_MI355_BF16: return XLLM_ROT(XLLM_MI355_BF16);
    case XLLM_MI355_FP16: return XLLM_ROT(XLLM_MI355_FP16);
    default: return XLLM_MI355_EDTYPE;
  }
#undef XLLM_ROT
}

// ---- MLA prologue --------------------------------------------------------------------------------------------------

constexpr int kLatent = 512, kRopeDim = 64;   // the widths that the MLA decode reads

struct MlaPrologueArgs {
  const uint16_t* q;
  uint16_t* q_out;
  const uint16_t* kv;
  uint16_t* kv_out;          // or null
  const uint16_t* weight;
  const char* cos_sin;
  const int64_t* positions;
  uint16_t* cache;           // or null
  const int32_t* slots;
  int64_t n_tokens, n_positions, n_slots;
  int64_t q_token, q_head, q_out_token, q_out_head, kv_row, kv_out_row;
  int64_t q_units;           // lanes of the query part
  int heads;
  int kv_blocks;             // workgroups of the latent part, the first ones of the grid
  float eps;
};

// The first kv_blocks workgroups take the tokens' latent rows, one wavefront per row: eight latent values per lane (one
// 16-byte word), their sum of squares over the wavefront, and the rope part in lanes 0-3.  The others rotate the rope
// part of the query heads, four lanes per head.  Bound by the bytes: 4099 tokens of 128 heads (149 MB, nearly all of it
// the heads' rope parts in rows of 128 bytes) 24.5 us = 6.1 TB/s.
template <int DT, int CT, bool INTERLEAVE>
__global__ __launch_bounds__(kRotThreads) void mla_prologue_kernel(MlaPrologueArgs a) {
  constexpr int kUnits = kRopeDim / 16;
  if (static_cast<int>(blockIdx.x) < a.kv_blocks) {
    const int64_t token = static_cast<int64_t>(blockIdx.x) * (kRotThreads / kWave) + threadIdx.x / kWave;
    const int lane = threadIdx.x & (kWave - 1);
    if (token >= a.n_tokens) return;
    const uint16_t* row = a.kv + token * a.kv_row;
    Pack<DT, 8> x, w, ra, rb;
    x.load(row + lane * 8);
    w.load(a.weight + lane * 8);
    const int unit = lane & (kUnits - 1);
    const int da = kLatent + (INTERLEAVE ? unit * 16 : unit * 8);
    const int db = kLatent + (INTERLEAVE ? unit * 16 + 8 : unit * 8 + kRopeDim / 2);
    ra.load(row + da);
    rb.load(row + db);
    const int64_t pos = a.positions[token];
    const bool turn = pos >= 0 && pos < a.n_positions;
    float c[8], s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      c[j] = 1.0f;
      s[j] = 0.0f;
    }
    if (turn) rot_row<CT, 8, true>(a.cos_sin, pos, kRopeDim, unit * 8, c, s);
    const int64_t slot = a.cache != nullptr ? a.slots[token] : -1;
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += x.get(j) * x.get(j);
    ss = group_sum<32>(ss);
    ss += __shfl_xor(ss, 32, kWave);
    const float r = 1.0f / __builtin_sqrtf(ss * (1.0f / kLatent) + a.eps);
#pragma unroll
    for (int j = 0; j < 4; ++j) x.put2(j, x.get(2 * j) * r * w.get(2 * j), x.get(2 * j + 1) * r * w.get(2 * j + 1));
    if (turn) turn_words<DT, 8, INTERLEAVE>(ra, rb, c, s);
    if (a.kv_out != nullptr) {
      uint16_t* o = a.kv_out + token * a.kv_out_row;
      x.store(o + lane * 8);
      if (lane < kUnits) {
        ra.store(o + da);
        rb.store(o + db);
      }
    }
    if (slot >= 0 && slot < a.n_slots) {
      uint16_t* o = a.cache + slot * (kLatent + kRopeDim);
      x.store(o + lane * 8);
      if (lane < kUnits) {
        ra.store(o + da);
        rb.store(o + db);
      }
    }
    return;
  }
  const int64_t idx = static_cast<int64_t>(blockIdx.x - a.kv_blocks) * kRotThreads + threadIdx.x;
  if (idx >= a.q_units) return;
  const int unit = static_cast<int>(idx & (kUnits - 1));
  const int64_t rest = idx / kUnits;
  const int64_t token = a.q_units <= 0x7fffffffLL ? static_cast<u32>(rest) / static_cast<u32>(a.heads) : rest / a.heads;
  const int head = static_cast<int>(rest - token * a.heads);
  const int da = INTERLEAVE ? unit * 16 : unit * 8;
  const int db = INTERLEAVE ? unit * 16 + 8 : unit * 8 + kRopeDim / 2;
  const uint16_t* in = a.q + token * a.q_token + head * a.q_head;
  uint16_t* out = a.q_out + token * a.q_out_token + head * a.q_out_head;
  Pack<DT, 8> x, y;
  x.load(in + da);
  y.load(in + db);
  const int64_t pos = a.positions[token];
  if (pos >= 0 && pos < a.n_positions) {
    float c[8], s[8];
    rot_row<CT, 8, true>(a.cos_sin, pos, kRopeDim, unit * 8, c, s);
    turn_words<DT, 8, INTERLEAVE>(x, y, c, s);
  }
  x.store(out + da);
  y.store(out + db);
}

template <int DT, int CT, bool INTERLEAVE>
int launch_mla_prologue(MlaPrologueArgs a, hipStream_t stream) {
  a.q_units = a.n_tokens * a.heads * (kRopeDim / 16);
  const int64_t kv = (a.n_tokens + kRotThreads / kWave - 1) / (kRotThreads / kWave);
  const int64_t groups = kv + (a.q_units + kRotThreads - 1) / kRotThreads;
  if (groups > kRotGroups) return XLLM_MI355_ESHAPE;
  a.kv_blocks = static_cast<int>(kv);
  mla_prologue_kernel<DT, CT, INTERLEAVE><<<dim3(static_cast<unsigned>(groups)), kRotThreads, 0, stream>>>(a);
  return static_cast<int>(hipGetLastError());
}

template <int DT>
int dispatch_mla_prologue(const MlaPrologueArgs& a, int interleave, int cos_sin_dtype, hipStream_t stream) {
#define XLLM_MLA_P(CT)                                                        \
  (interleave != 0 ? launch_mla_prologue<DT, CT, true>(a, stream)             \
                   : launch_mla_prologue<DT, CT, false>(a, stream))
  switch (cos_sin_dtype) {
    case XLLM_MI355_FP32: return XLLM_MLA_P(XLLM_MI355_FP32);
    case XLLM_MI355_BF16: return XLLM_MLA_P(XLLM_MI355_BF16);
    case XLLM_MI355_FP16: return XLLM_MLA_P(XLLM_MI355_FP16);
    default: return XLLM_MI355_EDTYPE;
  }
#undef XLLM_MLA_P
}

// Rows of `inner` elements at n0 strides of s0 and n1 strides of s1: does each lie apart from the others?
bool rows_apart(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t inner) {
  return ((n1 == 1 || s1 >= inner) && (n0 == 1 || s0 >= (n1 - 1) * s1 + inner)) ||
         ((n0 == 1 || s0 >= inner) && (n1 == 1 || s1 >= (n0 - 1) * s0 + inner));
}
bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace

int rope_cos_sin(const double* inv_freq, const int64_t* positions, int64_t first_position, int64_t n_rows, int64_t half,
                 double factor, void* out, int out_dtype, hipStream_t stream) {
  if (n_rows == 0) return XLLM_MI355_OK;
  if (inv_freq == nullptr || out == nullptr || n_rows < 0 || half <= 0) return XLLM_MI355_EINVAL;
  if (half > 4096 || n_rows > (1LL << 40)) return XLLM_MI355_ESHAPE;
  if (out_dtype != XLLM_MI355_FP32 && out_dtype != XLLM_MI355_BF16 && out_dtype != XLLM_MI355_FP16) return XLLM_MI355_EDTYPE;
  const Span w(out, n_rows * half * (out_dtype == XLLM_MI355_FP32 ? 8 : 4));
  if (w.meets(Span(inv_freq, half * 8)) || w.meets(Span(positions, n_rows * 8))) return XLLM_MI355_EINVAL;
  switch (out_dtype) {
    case XLLM_MI355_FP32: return launch_cos_sin<XLLM_MI355_FP32>(inv_freq, positions, first_position, n_rows, half, factor, out, stream);
    case XLLM_MI355_BF16: return launch_cos_sin<XLLM_MI355_BF16>(inv_freq, positions, first_position, n_rows, half, factor, out, stream);
    case XLLM_MI355_FP16: return launch_cos_sin<XLLM_MI355_FP16>(inv_freq, positions, first_position, n_rows, half, factor, out, stream);
    default: return XLLM_MI355_EDTYPE;
  }
}

int rotary_embedding(const int64_t* positions, const void* cos_sin, int64_t n_positions, const void* q, void* q_out,
                     const void* k, void* k_out, int64_t n_tokens, int64_t n_heads_q, int64_t n_heads_k,
                     int64_t head_dim_q, int64_t head_dim_k, int64_t rotary_offset_q, int64_t rotary_offset_k,
                     int64_t rotary_dim, const int64_t* q_strides, const int64_t* q_out_strides,
                     const int64_t* k_strides, const int64_t* k_out_strides, int interleave, int inverse, int dtype,
                     int cos_sin_dtype, hipStream_t stream) {
  if (n_tokens == 0) return XLLM_MI355_OK;
  if (positions == nullptr || cos_sin == nullptr || q == nullptr || q_out == nullptr || q_strides == nullptr ||
      q_out_strides == nullptr || n_tokens < 0 || n_positions <= 0 || n_heads_q <= 0 || n_heads_k < 0)
    return XLLM_MI355_EINVAL;
  if (n_heads_k > 0 && (k == nullptr || k_out == nullptr || k_strides == nullptr || k_out_strides == nullptr))
    return XLLM_MI355_EINVAL;
  if (dtype != XLLM_MI355_BF16 && dtype != XLLM_MI355_FP16 && dtype != XLLM_MI355_FP32) return XLLM_MI355_EDTYPE;
  if (cos_sin_dtype != XLLM_MI355_BF16 && cos_sin_dtype != XLLM_MI355_FP16 && cos_sin_dtype != XLLM_MI355_FP32)
    return XLLM_MI355_EDTYPE;
  if (n_heads_q > 65535 || n_heads_k > 65535 || head_dim_q > 65536 || head_dim_k > 65536 || n_tokens > (1LL << 31))
    return XLLM_MI355_ESHAPE;
  if (rotary_dim <= 0 || rotary_dim % 2 != 0 || rotary_offset_q < 0 || rotary_offset_q + rotary_dim > head_dim_q)
    return XLLM_MI355_ESHAPE;
  if (n_heads_k > 0 && (rotary_offset_k < 0 || rotary_offset_k + rotary_dim > head_dim_k)) return XLLM_MI355_ESHAPE;
  const int64_t es = dtype == XLLM_MI355_FP32 ? 4 : 2;
  const int64_t word = 16 / es;   // elements of 16 bytes
  const int64_t table_size = cos_sin_dtype == XLLM_MI355_FP32 ? 4 : 2;
  RotArgs a = {};
  auto side = [&](RotSide& s, const void* in, void* out, const int64_t* si, const int64_t* so, int64_t heads, int64_t dim,
                  int64_t offset) {
    s.in = static_cast<const char*>(in);
    s.out = static_cast<char*>(out);
    s.in_token = si[0];
    s.in_head = si[1];
    s.out_token = so[0];
    s.out_head = so[1];
    s.heads = static_cast<int>(heads);
    s.dim = static_cast<int>(dim);
    s.offset = static_cast<int>(offset);
    return !(si[0] < 0 || si[1] < 0 || so[0] < 0 || so[1] < 0);
  };
  bool copy_rest = false;
  // 16 bytes per lane where every word of every head starts on one; element by element otherwise
  bool vec = aligned(cos_sin, 16) && (rotary_dim / 2) % word == 0 && (rotary_dim / 2 * table_size) % 16 == 0;
  auto add = [&](RotSide& s) {
    vec = vec && aligned(s.in, 16) && aligned(s.out, 16) && s.in_token % word == 0 && s.in_head % word == 0 &&
          s.out_token % word == 0 && s.out_head % word == 0 && s.offset % word == 0 && s.dim % word == 0;
    copy_rest = copy_rest || (s.in != s.out && s.dim > rotary_dim);
  };
  if (!side(a.q, q, q_out, q_strides, q_out_strides, n_heads_q, head_dim_q, rotary_offset_q)) return XLLM_MI355_EINVAL;
  add(a.q);
  if (n_heads_k > 0) {
    if (!side(a.k, k, k_out, k_strides, k_out_strides, n_heads_k, head_dim_k, rotary_offset_k)) return XLLM_MI355_EINVAL;
    add(a.k);
  }
  // A result goes to its own operand, element for element, or apart from everything that is read, and the two results lie
  // apart; so do the heads of each.
  auto region = [&](const RotSide& s, bool out) {
    if (s.heads == 0) return Region{};
    return out ? Region{s.out, n_tokens, s.out_token * es, s.heads, s.out_head * es, s.dim * es}
               : Region{s.in, n_tokens, s.in_token * es, s.heads, s.in_head * es, s.dim * es};
  };
  for (const RotSide* s : {&a.q, &a.k}) {
    if (s->heads == 0) continue;
    const RotSide& other = s == &a.q ? a.k : a.q;
    if (!rows_apart(n_tokens, s->out_token, s->heads, s->out_head, s->dim)) return XLLM_MI355_EINVAL;
    const Region w = region(*s, true);
    if (s->in == s->out ? s->in_token != s->out_token || s->in_head != s->out_head : w.meets(region(*s, false)))
      return XLLM_MI355_EINVAL;
    if (w.meets(region(other, false)) || w.meets(region(other, true)) || w.span().meets(Span(positions, n_tokens * 8)) ||
        w.span().meets(Span(cos_sin, n_positions * rotary_dim * table_size)))
      return XLLM_MI355_EINVAL;
  }
  a.positions = positions;
  a.cos_sin = static_cast<const char*>(cos_sin);
  a.n_positions = n_positions;
  a.rot = static_cast<int>(rotary_dim);
  switch (dtype) {
    case XLLM_MI355_BF16: return dispatch_rotary<XLLM_MI355_BF16>(a, cos_sin_dtype, interleave, vec, copy_rest, inverse, n_tokens, stream);
    case XLLM_MI355_FP16: return dispatch_rotary<XLLM_MI355_FP16>(a, cos_sin_dtype, interleave, vec, copy_rest, inverse, n_tokens, stream);
    default: return dispatch_rotary<XLLM_MI355_FP32>(a, cos_sin_dtype, interleave, vec, copy_rest, inverse, n_tokens, stream);
  }
}

int mla_norm_rope_and_cache(const void* q_pe, void* q_pe_out, const void* kv, void* kv_out, const void* kv_weight, float eps,
                            const void* cos_sin, int64_t n_positions, const int64_t* positions, void* k_cache,
                            const int32_t* slots, int64_t n_tokens, int64_t n_heads, int64_t d_latent, int64_t d_rope,
                            int64_t q_token_stride, int64_t q_head_stride, int64_t q_out_token_stride,
                            int64_t q_out_head_stride, int64_t kv_row_stride, int64_t kv_out_row_stride,
                            int64_t block_size, int64_t num_blocks, int interleave, int dtype, int cos_sin_dtype,
                            hipStream_t stream) {
  if (n_tokens == 0) return XLLM_MI355_OK;
  if (q_pe == nullptr || q_pe_out == nullptr || kv == nullptr || kv_weight == nullptr || cos_sin == nullptr ||
      positions == nullptr || n_tokens < 0 || n_heads <= 0 || n_positions <= 0 || !(eps >= 0.0f))
    return XLLM_MI355_EINVAL;
  if (k_cache == nullptr && kv_out == nullptr) return XLLM_MI355_EINVAL;
  if (dtype != XLLM_MI355_BF16 && dtype != XLLM_MI355_FP16) return XLLM_MI355_EDTYPE;
  if (cos_sin_dtype != XLLM_MI355_BF16 && cos_sin_dtype != XLLM_MI355_FP16 && cos_sin_dtype != XLLM_MI355_FP32)
    return XLLM_MI355_EDTYPE;
  if (d_latent != kLatent || d_rope != kRopeDim || n_heads > 65535 || n_tokens > (1LL << 31)) return XLLM_MI355_ESHAPE;
  if (q_token_stride < 0 || q_head_stride < 0 || q_out_token_stride < 0 || q_out_head_stride < 0 ||
      kv_row_stride < d_latent + d_rope || (kv_out != nullptr && kv_out_row_stride < d_latent + d_rope))
    return XLLM_MI355_EINVAL;
  if (k_cache != nullptr) {
    if (slots == nullptr || block_size <= 0 || num_blocks <= 0) return XLLM_MI355_EINVAL;
    if (block_size > 0x7fffffffLL || num_blocks > 0x7fffffffLL || block_size * num_blocks > 0x7fffffffLL)
      return XLLM_MI355_ESHAPE;
  }
  if (!aligned(q_pe, 16) || !aligned(q_pe_out, 16) || !aligned(kv, 16) || !aligned(kv_out, 16) || !aligned(kv_weight, 16) ||
      !aligned(cos_sin, 16) || !aligned(k_cache, 16) ||
      ((q_token_stride | q_head_stride | q_out_token_stride | q_out_head_stride | kv_row_stride) & 7) != 0 ||
      (kv_out != nullptr && (kv_out_row_stride & 7) != 0))
    return XLLM_MI355_EALIGN;
  {
    const int64_t table_size = cos_sin_dtype == XLLM_MI355_FP32 ? 4 : 2, row = kLatent + kRopeDim;
    const Region sq{q_pe, n_tokens, q_token_stride * 2, n_heads, q_head_stride * 2, kRopeDim * 2};
    const Region skv{kv, n_tokens, kv_row_stride * 2, 1, 0, row * 2};
    const Span rest[4] = {Span(kv_weight, kLatent * 2), Span(cos_sin, n_positions * kRopeDim * table_size),
                          Span(positions, n_tokens * 8), Span(slots, k_cache != nullptr ? n_tokens * 4 : 0)};
    const Region wq{q_pe_out, n_tokens, q_out_token_stride * 2, n_heads, q_out_head_stride * 2, kRopeDim * 2};
    const Region wkv = kv_out != nullptr ? Region{kv_out, n_tokens, kv_out_row_stride * 2, 1, 0, row * 2} : Region{};
    const Region wc = k_cache != nullptr ? Region{k_cache, 1, 0, 1, 0, num_blocks * block_size * row * 2} : Region{};
    if (!rows_apart(n_tokens, q_out_token_stride, n_heads, q_out_head_stride, kRopeDim)) return XLLM_MI355_EINVAL;
    if (q_pe_out == q_pe ? q_out_token_stride != q_token_stride || q_out_head_stride != q_head_stride : wq.meets(sq))
      return XLLM_MI355_EINVAL;
    if (kv_out == kv ? kv_out_row_stride != kv_row_stride : wkv.meets(skv)) return XLLM_MI355_EINVAL;
    if (wq.meets(skv) || wkv.meets(sq) || wq.meets(wkv)) return XLLM_MI355_EINVAL;
    if (wc.meets(sq) || wc.meets(skv) || wc.meets(wq) || wc.meets(wkv)) return XLLM_MI355_EINVAL;
    for (const Span& r : rest)
      if (wq.span().meets(r) || (kv_out != nullptr && wkv.span().meets(r)) || (k_cache != nullptr && wc.span().meets(r)))
        return XLLM_MI355_EINVAL;
  }
  MlaPrologueArgs a = {};
  a.q = static_cast<const uint16_t*>(q_pe);
  a.q_out = static_cast<uint16_t*>(q_pe_out);
  a.kv = static_cast<const uint16_t*>(kv);
  a.kv_out = static_cast<uint16_t*>(kv_out);
  a.weight = static_cast<const uint16_t*>(kv_weight);
  a.cos_sin = static_cast<const char*>(cos_sin);
  a.positions = positions;
  a.cache = static_cast<uint16_t*>(k_cache);
  a.slots = slots;
  a.n_tokens = n_tokens;
  a.n_positions = n_positions;
  a.n_slots = k_cache != nullptr ? block_size * num_blocks : 0;
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.q_out_token = q_out_token_stride;
  a.q_out_head = q_out_head_stride;
  a.kv_row = kv_row_stride;
  a.kv_out_row = kv_out_row_stride;
  a.heads = static_cast<int>(n_heads);
  a.eps = eps;
  return dtype == XLLM_MI355_BF16 ? dispatch_mla_prologue<XLLM_MI355_BF16>(a, interleave, cos_sin_dtype, stream)
                                  : dispatch_mla_prologue<XLLM_MI355_FP16>(a, interleave, cos_sin_dtype, stream);
}

}  // namespace xllm_mi355
