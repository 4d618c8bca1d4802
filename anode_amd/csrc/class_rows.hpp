// Shared by the operators over rows of many classes (top_k.hip, distill.hip, verify_draft.hip): the element types of
// the logits, a row as 16-byte groups, the running maximum and sum of a softmax, and the argument checks.
#pragma once

#include "common.hpp"

#include <cmath>
#include <tuple>

namespace anode {

// C ABI element type -> device element type.  bfloat16 and half arrays are declared as uint16_t in the header.
typedef __bf16 bf16_t;
typedef _Float16 f16_t;

constexpr uint32_t kNoClass = 0xffffffffu;  // "no class": the index of an empty slot, a token that was not drawn
constexpr uint32_t kMaxSlots = 1024;        // largest k of the top-k and distillation entry points

// The refusals of these entry points: nothing is enqueued, the reason goes to stderr and the code to
// anode_gpu_take_last_error(), and the entry point returns it.
static inline int refuse(const char *symbol, const char *what) {
  note_error(symbol, hipErrorInvalidValue, what);
  return int(hipErrorInvalidValue);
}

// acquire_scratch() with the code of its own failure, 0 if there was none (runtime.hip).  (What the process recorded last may be
// another thread's error, or taken by it.)
ScratchLease acquire_scratch(hipStream_t stream, size_t bytes, const char *symbol, int &error);
// What note_launch() does, of a launch whose own result is known: `e` is recorded and printed if it is an error, and returned.
// (The thread's error state may hold an error from before, or the same one from an earlier launch.)
int note_launched(const char *symbol, hipError_t e);

// The stream's scratch (runtime.hip) for these entry points, which return an error code and let no exception out: ptr is
// null when it cannot be had, and `error` then what the entry point returns.
struct RowsScratch {
  ScratchLease lease;
  int error;
};
static inline RowsScratch rows_scratch(hipStream_t stream, size_t bytes, const char *symbol) {
  RowsScratch s = {ScratchLease{}, 0};
  try {
    s.lease = acquire_scratch(stream, bytes, symbol, s.error);
  } catch (...) {
    note_error(symbol, hipErrorOutOfMemory, "cannot keep account of the scratch");
    s.error = int(hipErrorOutOfMemory);
  }
  return s;
}
// The scratch that each of them needs for [classes, rows] (distill.hip, top_k.hip, verify_draft.hip).
size_t distill_scratch(uint32_t classes, uint32_t rows);
size_t top_k_scratch(uint32_t classes, uint32_t rows, uint32_t k);
size_t verify_scratch(uint32_t classes, uint32_t sequences);

// What the row entry points ask of their scalars; 0 when they are fine.  The checks come before any device call.
static inline int check_rows(const char *symbol, uint32_t classes, uint32_t stride, uint32_t k, float temperature) {
  if (stride != 0u && stride < classes) return refuse(symbol, "the stride is shorter than a row (0 = rows without padding)");
  if (k > kMaxSlots) return refuse(symbol, "more than 1024 slots a row");
  if (!(temperature > 0.0f) || !std::isfinite(temperature) || !std::isfinite(1.4426950408889634 / double(temperature)) ||
      !std::isfinite(float(1.4426950408889634 / double(temperature)))) {
    return refuse(symbol, "the temperature is not a positive finite number");
  }
  return 0;
}

template <typename T>
static inline bool misaligned(const T *p) {
  return (reinterpret_cast<uintptr_t>(p) & (alignof(T) - 1u)) != 0;
}

#if defined(__HIPCC__)

// Launches a kernel with a workgroup an item, or as many as a launch takes, and returns how that went, which <<< >>> does not tell.
// (HIP refuses 2^32 work-items and more: 2^24 workgroups of 256.  The kernels here take the further items in turn.)
template <typename... P, typename... A>
static inline hipError_t launch(void (*kernel)(P...), uint64_t items, uint32_t threads, size_t lds, hipStream_t stream, A... args) {
  const uint64_t most = (uint64_t(1) << 31) / threads;
  const uint32_t grid = uint32_t(items < most ? items : most);
  std::tuple<P...> values(args...);  // of the kernel's own parameter types
  return std::apply(
      [&](P &...p) {
        void *at[] = {const_cast<void *>(static_cast<const void *>(&p))...};
        return hipLaunchKernel(reinterpret_cast<const void *>(kernel), dim3(grid), dim3(threads), at, lds, stream);
      },
      values);
}

constexpr float kMinusInf = -__builtin_huge_valf();

// Moves between lanes without the LDS pipe (data-parallel primitives): the value of the lane 1, 2, 4 or 8 before in its
// row of sixteen, of the last lane of the row before (rows 1 and 3), or of lane 31 (rows 2 and 3); lanes that get none keep
// `none`.  Six such steps make lane 63 the sum of all lanes, and every lane the sum of those up to it, in about 100
// clocks, where six exchanges through ds_bpermute take about 600 (a double is two of them).
template <int STEP>
__device__ inline uint32_t lane_before(uint32_t none, uint32_t v) {
  constexpr int kControl = STEP < 4 ? 0x110 + (1 << STEP) : STEP == 4 ? 0x142 : 0x143;  // row_shr 1 2 4 8, row_bcast 15 31
  constexpr int kRows = STEP < 4 ? 0xf : STEP == 4 ? 0xa : 0xc;
  return uint32_t(__builtin_amdgcn_update_dpp(int(none), int(v), kControl, kRows, 0xf, false));
}
template <int STEP>
__device__ inline float lane_before(float none, float v) {
  return __uint_as_float(lane_before<STEP>(__float_as_uint(none), __float_as_uint(v)));
}
template <int STEP>
__device__ inline double lane_before(double none, double v) {
  const uint64_t n = __builtin_bit_cast(uint64_t, none), b = __builtin_bit_cast(uint64_t, v);
  const uint64_t lo = lane_before<STEP>(uint32_t(n), uint32_t(b)), hi = lane_before<STEP>(uint32_t(n >> 32), uint32_t(b >> 32));
  return __builtin_bit_cast(double, hi << 32 | lo);
}
// A lane's value in every lane (the lane is the same in all of them).
__device__ inline uint32_t from_lane(uint32_t v, int lane) { return uint32_t(__builtin_amdgcn_readlane(int(v), lane)); }
__device__ inline float from_lane(float v, int lane) { return __uint_as_float(from_lane(__float_as_uint(v), lane)); }
__device__ inline double from_lane(double v, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, uint64_t(from_lane(uint32_t(b >> 32), lane)) << 32 | from_lane(uint32_t(b), lane));
}
// Sum over the lanes up to this one.
template <typename V>
__device__ inline V lanes_upto(V v) {
  v += lane_before<0>(V(0), v);
  v += lane_before<1>(V(0), v);
  v += lane_before<2>(V(0), v);
  v += lane_before<3>(V(0), v);
  v += lane_before<4>(V(0), v);
  v += lane_before<5>(V(0), v);
  return v;
}
template <typename V>
__device__ inline V lanes_sum(V v) {
  return from_lane(lanes_upto(v), kWave - 1);
}

// The largest of the lanes' values, the same in every lane.
__device__ inline float lanes_max(float v) {
  v = fmaxf(v, lane_before<0>(v, v));
  v = fmaxf(v, lane_before<1>(v, v));
  v = fmaxf(v, lane_before<2>(v, v));
  v = fmaxf(v, lane_before<3>(v, v));
  v = fmaxf(v, lane_before<4>(v, v));
  v = fmaxf(v, lane_before<5>(v, v));
  return __shfl(v, kWave - 1, kWave);
}

// One 16-byte group of a row: W values.
template <typename T>
struct Group {
  static constexpr int W = 16 / int(sizeof(T));
};

__device__ inline void unpack(const u32x4 &q, float (&v)[4], const float *) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(q[i]);
}
__device__ inline void unpack(const u32x4 &q, float (&v)[8], const bf16_t *) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(q[i] << 16);
    v[2 * i + 1] = __uint_as_float(q[i] & 0xffff0000u);
  }
}
__device__ inline void unpack(const u32x4 &q, float (&v)[8], const f16_t *) {
  typedef f16_t f16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t word = q[i];  // (a copy: the bit cast of a vector's element itself reads element 0)
    const f16x2 h = __builtin_bit_cast(f16x2, word);
    v[2 * i] = float(h.x);
    v[2 * i + 1] = float(h.y);
  }
}

// One value.  (Of a conversion from bfloat16 the compiler takes it that no signalling NaN comes out, but it is a shift.)
__device__ inline float widened(float x) { return x; }
__device__ inline float widened(f16_t x) { return float(x); }
__device__ inline float widened(bf16_t x) { return __uint_as_float(uint32_t(__builtin_bit_cast(uint16_t, x)) << 16); }

// Rounding to the element type: to nearest, ties to even (the conversions of gfx950).
__device__ inline u32x4 pack(const float (&v)[4], const float *) {
  return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
}
template <typename T>
__device__ inline u32x4 pack(const float (&v)[8], const T *) {
  typedef T x2 __attribute__((ext_vector_type(2)));
  u32x4 q;
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = __builtin_bit_cast(uint32_t, x2{T(v[2 * i]), T(v[2 * i + 1])});
  return q;
}

// A row's values in 16-byte groups from its start: group g holds the values g * W ... g * W + W - 1 of the row's `n`, those of
// them that exist.  (A 16-byte load needs no alignment beyond the element's.)
template <typename T>
struct RowGroups {
  static constexpr int W = Group<T>::W;
  uint32_t n, groups;
  __device__ explicit RowGroups(uint32_t n_) : n(n_), groups(n_ / uint32_t(W) + (n_ % uint32_t(W) != 0u)) {}
  __device__ uint32_t first(uint32_t g) const { return g * uint32_t(W); }
  __device__ bool whole(uint32_t g) const { return g < n / uint32_t(W); }
};

// 16-byte groups through a buffer descriptor: one offset register serves every group of a thread (the rest of the address
// is scalar), a group past the end loads zeros and stores nothing.  The memory has to be 4-byte aligned and shorter than
// 4 GiB.  NT: kNtStore as in store_stream().
struct GroupBuffer {
  __amdgpu_buffer_rsrc_t rsrc;
  template <typename T>
  __device__ GroupBuffer(const T *p, uint32_t groups)
      : rsrc(__builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(p), 0, int(groups * 16u), 0x00027000)) {}
  __device__ u32x4 load(uint32_t thread_bytes, uint32_t bytes) const {
    return __builtin_amdgcn_raw_buffer_load_b128(rsrc, int(thread_bytes), int(bytes), 0);
  }
  template <int NT>
  __device__ void store(u32x4 v, uint32_t thread_bytes, uint32_t bytes) const {
    __builtin_amdgcn_raw_buffer_store_b128(v, rsrc, int(thread_bytes), int(bytes), (NT & kNtStore) != 0 ? 18 : 0);
    // A write to the data registers of such a store right behind it has changed the stored value here; the compiler, which
    // keeps the distance after other stores of more than 8 bytes, takes none to be needed where the offset is scalar.
    asm volatile("s_nop 1" ::"v"(v) : "memory");
  }
};

// The values of group g; those that are not the row's are `fill` and are not read.
template <typename T>
__device__ inline void load_group(const RowGroups<T> &rg, const T *row, uint32_t g, float fill, float (&v)[Group<T>::W]) {
  constexpr int W = Group<T>::W;
  if (rg.whole(g)) {
    unpack(load_stream<0, int(sizeof(T))>(reinterpret_cast<const u32x4 *>(row + rg.first(g))), v, row);
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = rg.first(g) + uint32_t(j) < rg.n ? float(row[rg.first(g) + uint32_t(j)]) : fill;
  }
}

// A whole group to where the row has it; NT (kNtStore): past the caches, for groups that lie on 16-byte boundaries.
template <int NT, int ALIGN, typename V>
__device__ inline void store_group(void *p, V v) {
  if constexpr ((NT & kNtStore) != 0) {
    store_stream<NT>(static_cast<V *>(p), v);
  } else {
    typedef V VU __attribute__((aligned(ALIGN)));
    *reinterpret_cast<VU *>(p) = v;
  }
}

// ---- statistics of a row: its maximum m and S = sum of exp((x - m) / T) = sum of exp2((x - m) * c) ----
//
// The fast form spends one fused multiply-add on a value's exponent: exp2(x * c - R) with R = fl(b * c) for a running
// reference b >= the values seen.  R's rounding is a factor common to all terms, which true_sum() takes out again at the
// end.  b starts at -limit, limit = 65536 / c: while it stays inside (-limit, limit) R is off by less than 2^-8 and
// nothing overflows, whatever single values hold (-inf and the lowest value of a type add 0, a NaN shows in S).  A
// row whose maximum lies outside -- nothing but -inf or a mask's lowest values, +inf, or values without measure --
// is summed again in the plain form, exp2((x - m) * c); of rows in earnest those are the positions that a mask empties.
struct Scale {
  float c, limit;
};
static inline Scale scale_for(float temperature) {
  const double c = 1.4426950408889634 / double(temperature);
  const double limit = 65536.0 / c;
  return Scale{float(c), float(limit < 1e38 ? limit : 1e38)};
}

struct SoftmaxSum {
  float m, s;
};

// The larger of two, and the largest of m and the values, two values an instruction; NaN where one of them is a NaN, of either
// kind.  (fmaxf() passes over a quiet NaN only: it quiets a signalling one by an instruction a value, and not at all one that was
// widened from bfloat16.  Of a signalling NaN and a number the hardware's maximum makes a quiet NaN, which the next one passes
// over, and the number is lost.)
__device__ inline float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }
template <int COUNT>
__device__ inline float max_of(float m, const float (&v)[COUNT]) {
  static_assert(COUNT == 2 || COUNT % 4 == 0, "values are taken four at a time");
  // (written out, the two of a step side by side: left to the compiler the held rows of distill.hip spill three registers more)
  if constexpr (COUNT == 2) {
    asm("v_maximum3_f32 %0, %0, %1, %2" : "+v"(m) : "v"(v[0]), "v"(v[1]));
  } else {
#pragma unroll
    for (int j = 0; j < COUNT; j += 4) {
      asm("v_maximum3_f32 %0, %0, %1, %2\n\tv_maximum3_f32 %0, %0, %3, %4" : "+v"(m) : "v"(v[j]), "v"(v[j + 1]), "v"(v[j + 2]), "v"(v[j + 3]));
    }
  }
  return m;
}

// The fast form.
template <int COUNT>
__device__ inline void fold_below(SoftmaxSum &t, float m, const float (&v)[COUNT], float c) {  // m: the new reference, >= t.m and all values, or a NaN
  const float shift = m * c;
  if (m > t.m) {
    t.s *= __builtin_amdgcn_exp2f(t.m * c - shift);
    t.m = m;
  }
  float s[2] = {__builtin_amdgcn_exp2f(fmaf(v[0], c, -shift)), __builtin_amdgcn_exp2f(fmaf(v[1], c, -shift))};
#pragma unroll
  for (int j = 2; j < COUNT; ++j) s[j & 1] += __builtin_amdgcn_exp2f(fmaf(v[j], c, -shift));
  t.s += s[0] + s[1];
}
template <int COUNT>
__device__ inline void fold(SoftmaxSum &t, const float (&v)[COUNT], float c) {
  fold_below(t, max_of(t.m, v), v, c);
}
__device__ inline void fold_one(SoftmaxSum &t, float x, float c) {
  const float v[2] = {x, kMinusInf};
  fold(t, v, c);
}
// The lanes' parts together, the same in every lane of the wave, added in a fixed order: first the maximum of all, then each lane's
// sum about it.  (Merging pairs at every step takes two exponentials each.)
__device__ inline SoftmaxSum wave_merge(SoftmaxSum t, float c) {
  SoftmaxSum r = {lanes_max(t.m), 0.0f};
  r.s = lanes_upto(t.s * __builtin_amdgcn_exp2f(t.m * c - r.m * c));
  // (an exchange, not from_lane(): results in scalar registers push the held rows of distill.hip out of the vector ones)
  r.s = __shfl(r.s, kWave - 1, kWave);
  return r;
}
// COUNT <= 16 entries in LDS merged, the same in every lane.
template <int COUNT>
__device__ inline SoftmaxSum lane_merge(const SoftmaxSum *lds, float c) {
  static_assert(COUNT <= 16, "an entry a lane of a row of sixteen");
  const uint32_t lane = threadIdx.x & 15u;
  SoftmaxSum t = lds[lane < uint32_t(COUNT) ? lane : 0u];
  if (lane >= uint32_t(COUNT)) t.s = 0.0f;  // (an entry again, of which nothing is added)
  SoftmaxSum r = {t.m, 0.0f};
  r.m = fmaxf(r.m, lane_before<0>(r.m, r.m));
  r.m = fmaxf(r.m, lane_before<1>(r.m, r.m));
  r.m = fmaxf(r.m, lane_before<2>(r.m, r.m));
  r.m = fmaxf(r.m, lane_before<3>(r.m, r.m));
  r.m = __shfl(r.m, 15, 16);
  r.s = t.s * __builtin_amdgcn_exp2f(t.m * c - r.m * c);
  r.s += lane_before<0>(0.0f, r.s);
  r.s += lane_before<1>(0.0f, r.s);
  r.s += lane_before<2>(0.0f, r.s);
  r.s += lane_before<3>(0.0f, r.s);
  r.s = __shfl(r.s, 15, 16);
  return r;
}
// The same in every thread of the workgroup; `lds` holds one entry a wave.  Ends with a barrier.
template <int WAVES>
__device__ inline SoftmaxSum block_merge(SoftmaxSum t, float c, SoftmaxSum *lds) {
  t = wave_merge(t, c);
  if constexpr (WAVES > 1) {
    if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = t;
    __syncthreads();
    t = lane_merge<WAVES>(lds, c);
  }
  __syncthreads();
  return t;
}
// Whether the fast form holds for a row of this maximum.
__device__ inline bool measured(float m, Scale sc) { return fabsf(m) < sc.limit; }
// The same of both: a row with a NaN has a sum that is one, and its maximum may lack values that lay beside the NaN.
__device__ inline bool measured(SoftmaxSum t, Scale sc) { return measured(t.m, sc) && t.s == t.s; }
// The reference's rounding taken out: S about m itself.
__device__ inline float true_sum(SoftmaxSum t, float c) { return t.s * __builtin_amdgcn_exp2f(fmaf(-t.m, c, t.m * c)); }

// A row, or a part of one, as it is streamed: `head` single values, `groups` 16-byte groups, `tail` single values.  The
// single values are taken one a thread.  head = 0 for kernels that only read (a 16-byte load may start at any
// element); a kernel that stores takes as many as bring its groups to a 128-byte line of the output.
template <typename T>
struct RowSpan {
  static constexpr int W = Group<T>::W;
  uint32_t head, groups, tail;
  __device__ RowSpan(uint32_t n, uint32_t head_) : head(head_ < n ? head_ : n) {
    groups = (n - head) / uint32_t(W);
    tail = n - head - groups * uint32_t(W);
  }
  __device__ bool single(uint32_t thread) const { return thread < head + tail; }
  // the place of the thread's single value; 0 (any place) for a thread that has none
  __device__ uint32_t single_at(uint32_t thread) const {
    return thread < head ? thread : single(thread) ? thread + groups * uint32_t(W) : 0u;
  }
  __device__ uint32_t first(uint32_t g) const { return head + g * uint32_t(W); }
};

// Values from the start of `p` to the next 128-byte line.
template <typename T>
__device__ inline uint32_t values_to_line(const T *p) {
  return uint32_t((128u - (reinterpret_cast<uintptr_t>(p) & 127u)) & 127u) / uint32_t(sizeof(T));
}

// Makes the compiler forget what it knows of a group held in registers: values unpacked from it before would otherwise
// be kept beside it until they are asked for again.
__device__ inline void forget(u32x4 &q) { asm volatile("" : "+v"(q)); }

// U groups of a thread: g, g + THREADS, ...  A group past the end reads the last one again (a branch round each load
// would make every load wait for the one before, and a tile that is fetched ahead in a branch is waited for at its end: so
// the tile behind the last is fetched too).  There is at least one group.
template <typename T, int THREADS, int U>
__device__ inline void load_tile(const RowSpan<T> &span, const T *row, uint32_t g, u32x4 (&q)[U]) {
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t at = min(g + uint32_t(u) * uint32_t(THREADS), span.groups - 1u);
    q[u] = load_stream<0, int(sizeof(T))>(reinterpret_cast<const u32x4 *>(row + size_t(span.first(at))));
  }
}
template <typename T, int U>
__device__ inline void unpack_tile(const u32x4 (&q)[U], float (&v)[U * Group<T>::W]) {
  constexpr int W = Group<T>::W;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float w[W];
    unpack(q[u], w, static_cast<const T *>(nullptr));
#pragma unroll
    for (int j = 0; j < W; ++j) v[u * W + j] = w[j];
  }
}
template <typename T, int THREADS, int U>
__device__ inline void mask_tile(const RowSpan<T> &span, uint32_t g, float fill, float (&v)[U * Group<T>::W]) {
  constexpr int W = Group<T>::W;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const bool in = g + uint32_t(u) * uint32_t(THREADS) < span.groups;
#pragma unroll
    for (int j = 0; j < W; ++j) v[u * W + j] = in ? v[u * W + j] : fill;
  }
}

// The plain form, for rows that the fast one does not measure: two passes, U groups of a thread on their way together (the loss
// of 512 rows of 131072 bf16 at the type's lowest value 64 us, 26 of random values; value by value, and with one wave for
// rows in parts, it took 1205 and, of 4 rows, 562 instead of 12).  -inf only
// (or nothing): m = -inf, S = 0.  A NaN is ignored by m and makes S NaN; so does +inf.  A thread adds its groups' sums in
// 64 bits: a long row of a mask's lowest value is nothing but ones, of which 32 bits hold 2^24.
template <typename T, int THREADS, int U>
__device__ inline SoftmaxSum plain_stats(const T *row, uint32_t n, float c, float *lds) {
  constexpr int N = U * Group<T>::W;
  const RowSpan<T> span(n, 0u);
  SoftmaxSum t = {kMinusInf, 0.0f};
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    const float about = t.m == kMinusInf ? 0.0f : t.m;
    float top = kMinusInf;
    double sum = 0.0;
    if (span.single(threadIdx.x)) {  // (the tail: fewer than a group)
      const float x = widened(row[span.single_at(threadIdx.x)]);
      if (pass == 0) {
        top = x > top ? x : top;
      } else {
        sum = double(__builtin_amdgcn_exp2f((x - about) * c));
      }
    }
#pragma unroll 1
    for (uint32_t g = threadIdx.x; g < span.groups; g += uint32_t(THREADS) * uint32_t(U)) {
      u32x4 q[U];
      float v[N];
      load_tile<T, THREADS, U>(span, row, g, q);
      unpack_tile<T, U>(q, v);
      if (U > 1) mask_tile<T, THREADS, U>(span, g, kMinusInf, v);
      if (pass == 0) {
        // (a comparison that no NaN passes, of either kind: not a maximum)
#pragma unroll
        for (int j = 0; j < N; ++j) top = v[j] > top ? v[j] : top;
      } else {
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < N; ++j) s += __builtin_amdgcn_exp2f((v[j] - about) * c);
        sum += double(s);
      }
    }
    float v = pass == 0 ? top : float(sum);
#pragma unroll 1
    for (int off = kWave / 2; off > 0; off >>= 1) {
      const float o = __shfl_xor(v, off, kWave);
      v = pass == 0 ? fmaxf(v, o) : v + o;
    }
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll 1
    for (int w = 1; w < THREADS / kWave; ++w) v = pass == 0 ? fmaxf(v, lds[w]) : v + lds[w];
    if (pass == 0) {
      t.m = v;
    } else {
      t.s = v;
    }
  }
  __syncthreads();
  return t;
}

// A thread's running reference and sum over its part of a row (merge them with block_merge): tiles of U groups a thread,
// the next tile on its way while one is folded.
template <typename T, int THREADS, int U>
__device__ inline SoftmaxSum stream_stats(const RowSpan<T> &span, const T *row, Scale sc) {
  constexpr uint32_t kTile = uint32_t(THREADS) * uint32_t(U);
  SoftmaxSum st = {-sc.limit, 0.0f};
  // (the head can hold more values than a small workgroup has threads)
  for (uint32_t i = threadIdx.x; span.single(i); i += THREADS) fold_one(st, float(row[span.single_at(i)]), sc.c);
  if (span.groups != 0u) {
    u32x4 q[U];
    load_tile<T, THREADS, U>(span, row, threadIdx.x, q);
    for (uint32_t base = 0;; base += kTile) {
      float v[U * Group<T>::W];
      u32x4 next[U];
      const bool more = span.groups - base > kTile;
      load_tile<T, THREADS, U>(span, row, base + kTile + threadIdx.x, next);
      unpack_tile<T, U>(q, v);
      if (!more) mask_tile<T, THREADS, U>(span, base + threadIdx.x, kMinusInf, v);
      fold(st, v, sc.c);
      if (!more) break;
#pragma unroll
      for (int u = 0; u < U; ++u) q[u] = next[u];
    }
  }
  return st;
}

// The statistics of a row, or of a part of one, from its threads' parts, by the whole workgroup.  NORM: for a row's log-sum-exp
// alone, which is NaN whatever the maximum of a row with a NaN.
template <typename T, int THREADS, bool NORM>
__device__ inline SoftmaxSum finish_stats(SoftmaxSum t, const T *row, uint32_t n, Scale sc, SoftmaxSum *lds) {
  t = block_merge<THREADS / kWave>(t, sc.c, lds);
  if (NORM ? measured(t.m, sc) : measured(t, sc)) return SoftmaxSum{t.m, true_sum(t, sc.c)};
  return plain_stats<T, THREADS, (THREADS > kWave ? 2 : 1)>(row, n, sc.c, reinterpret_cast<float *>(lds));
}

// The statistics of the lanes' parts of a row together, the same in every lane; they are finished, whichever form they took, so
// no row is read again to join them.  (m = -inf, S = 0 for a lane that has none.)
__device__ inline SoftmaxSum join_lanes(SoftmaxSum t, float c) {
  SoftmaxSum r = {lanes_max(t.m), 0.0f};
  const float about = r.m == kMinusInf ? 0.0f : r.m;
  r.s = lanes_upto(t.s * __builtin_amdgcn_exp2f((t.m - about) * c));
  r.s = __shfl(r.s, kWave - 1, kWave);
  return r;
}

#endif  // __HIPCC__

}  // namespace anode
