// Shared by the operators over rows of many classes (top_k.hip, distill.hip, verify_draft.hip): the element types of
// the logits, a row as 16-byte groups, the running maximum and sum of a softmax, and the argument checks.
#pragma once

#include "common.hpp"

#include <cmath>

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

constexpr float kMinusInf = -__builtin_huge_valf();

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

// A row's values in 16-byte groups: group g holds the values g * W - shift ... g * W - shift + W - 1 of the row's
// `n`, those of them that exist.  Rows may start at any element: with shift = 0 the groups start where the row does
// (a 16-byte load needs no alignment beyond the element's); a kernel that stores chooses the shift so that its
// groups start on 16-byte boundaries of the output.
template <typename T>
struct RowGroups {
  static constexpr int W = Group<T>::W;
  uint32_t n, shift, groups;
  __device__ RowGroups(uint32_t n_, uint32_t shift_)
      : n(n_), shift(shift_), groups(uint32_t((uint64_t(n_) + shift_ + uint32_t(W) - 1u) / uint32_t(W))) {
    if (n_ == 0u) groups = 0u;
  }
  // index of the group's first value; wrapped below zero for the first group of a shifted row
  __device__ uint32_t first(uint32_t g) const { return g * uint32_t(W) - shift; }
  __device__ bool whole(uint32_t g) const {
    const uint64_t at = uint64_t(g) * uint32_t(W);
    return at >= shift && at + uint32_t(W) <= uint64_t(n) + shift;
  }
  __device__ bool has(uint32_t g, int j) const {
    const uint64_t at = uint64_t(g) * uint32_t(W) + uint32_t(j);
    return at >= shift && at < uint64_t(n) + shift;
  }
};

// The values of group g; those that are not the row's are `fill` and are not read.
template <typename T, int NT>
__device__ inline void load_group(const RowGroups<T> &rg, const T *row, uint32_t g, float fill, float (&v)[Group<T>::W]) {
  constexpr int W = Group<T>::W;
  if (rg.whole(g)) {
    unpack(load_stream<NT, int(sizeof(T))>(reinterpret_cast<const u32x4 *>(row + rg.first(g))), v, row);
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = rg.has(g, j) ? float(row[size_t(rg.first(g) + uint32_t(j))]) : fill;
  }
}

// A whole group to where the row has it, at any element.
template <int ALIGN, typename V>
__device__ inline void store_unaligned(void *p, V v) {
  typedef V VU __attribute__((aligned(ALIGN)));
  *reinterpret_cast<VU *>(p) = v;
}

// Maximum m and sum s of exp2((x - m) * c) over what has been seen; c = log2(e) / temperature.  The difference is
// taken before the product: values up to the type's largest and lowest neither overflow nor cancel.  Nothing seen,
// or -inf only: m = -inf and s = 0.  A NaN is ignored by m and makes s NaN; so does +inf.
struct SoftmaxSum {
  float m, s;
};
__device__ inline float exp_scaled(float x, float m, float c) { return __builtin_amdgcn_exp2f((x - m) * c); }
// exp2((m - to) * c) with 0 for a sum that holds nothing yet
__device__ inline float rescale(float m, float to, float c) { return m == kMinusInf ? 0.0f : exp_scaled(m, to, c); }
__device__ inline SoftmaxSum merge(SoftmaxSum a, SoftmaxSum b, float c) {
  SoftmaxSum r;
  r.m = fmaxf(a.m, b.m);
  r.s = a.s * rescale(a.m, r.m, c) + b.s * rescale(b.m, r.m, c);
  return r;
}

// Folds `count` values into the running maximum and sum.
template <int COUNT>
__device__ inline void fold(SoftmaxSum &t, const float (&v)[COUNT], float c) {
  float m = t.m;
#pragma unroll
  for (int j = 0; j < COUNT; ++j) m = fmaxf(m, v[j]);
  if (m != t.m) {
    t.s *= rescale(t.m, m, c);
    t.m = m;
  }
  const float about = m == kMinusInf ? 0.0f : m;  // (-inf minus 0 stays -inf and adds nothing; a NaN still shows)
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < COUNT; ++j) s += exp_scaled(v[j], about, c);
  t.s += s;
}

// Every thread of the workgroup gets the merged maximum and sum, merged in a fixed order: butterflies in the wave, then
// the waves in turn.  `lds` holds one entry a wave; the call ends with a barrier.
template <int WAVES>
__device__ inline SoftmaxSum block_merge(SoftmaxSum t, float c, SoftmaxSum *lds) {
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) {
    SoftmaxSum o;
    o.m = __shfl_xor(t.m, off, kWave);
    o.s = __shfl_xor(t.s, off, kWave);
    t = merge(t, o, c);
  }
  if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = t;
  __syncthreads();
  t = lds[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) t = merge(t, lds[w], c);
  __syncthreads();
  return t;
}

#endif  // __HIPCC__

}  // namespace anode
