// Distillation from a teacher's top logits: the loss of a row of student logits against the teacher's k largest
// logits of that row, and its gradient.  No kernel of the reference corresponds to it; it stands beside the row form
// of softmax + categorical NLL (softmax.hip), which is the case of one slot that holds all of the mass.
//
// With x the student's row, m = max x, S = sum exp((x - m) / T), q_j = exp((x_j - m) / T) / S, and the teacher's slots
// (t_k, i_k), of which those with i_k < classes and t_k > -inf count:
//   p_k = exp(t_k / T) / sum exp(t / T)          without the teacher's norm: the mass is 1 by definition
//   p_k = exp(t_k / T - log_norm)                with it: the slots hold the share that the teacher gave them
//   loss = sum p_k (ln p_k - ln q_{i_k})
//   d loss / d x_j = (P q_j - sum of the p_k with i_k = j) / T,   P = sum p_k
// The k terms of a row are computed in 64 bits: the loss is a small difference of large terms where the student is
// close, and they are few.
#include "class_rows.hpp"

#include <cmath>

namespace anode {
namespace {

struct Teacher {
  const float *value;
  const uint32_t *index;
  const float *log_norm;  // null: the slots are the whole distribution
  uint32_t k;
  __device__ bool counts(size_t at, uint32_t n) const { return index[at] < n && value[at] > kMinusInf; }
};

// What a wave needs of a row's teacher: probability of slot j is exp(value * inv_t - shift) * scale.
struct TeacherRow {
  double shift, scale, mass;
  bool any;
};

// By one whole wave; `first` is the row's first slot.
__device__ inline TeacherRow teacher_row(const Teacher &t, size_t row, uint32_t n, double inv_t) {
  const uint32_t lane = threadIdx.x & (kWave - 1);
  const size_t first = row * t.k;
  float top = kMinusInf;
  for (uint32_t j = lane; j < t.k; j += kWave) {
    if (t.counts(first + j, n)) top = fmaxf(top, t.value[first + j]);
  }
  top = wave_max(top);
  TeacherRow r;
  r.any = top > kMinusInf;
  r.shift = t.log_norm != nullptr ? double(t.log_norm[row]) : double(top) * inv_t;
  double sum = 0.0;
  for (uint32_t j = lane; j < t.k; j += kWave) {
    if (t.counts(first + j, n)) sum += exp(double(t.value[first + j]) * inv_t - r.shift);
  }
  sum = wave_sum(sum);
  r.scale = t.log_norm != nullptr ? 1.0 : 1.0 / sum;
  r.mass = t.log_norm != nullptr ? sum : 1.0;
  return r;
}

// The row's loss, by one whole wave.
template <typename T>
__device__ inline float row_loss(const Teacher &t, size_t row, const T *x, uint32_t n, SoftmaxSum st, double inv_t) {
  const uint32_t lane = threadIdx.x & (kWave - 1);
  const size_t first = row * t.k;
  const TeacherRow tr = teacher_row(t, row, n, inv_t);
  if (!tr.any) return 0.0f;
  const double log_s = log(double(st.s)), log_scale = log(tr.scale);
  double loss = 0.0;
  for (uint32_t j = lane; j < t.k; j += kWave) {
    if (!t.counts(first + j, n)) continue;
    const double lp = double(t.value[first + j]) * inv_t - tr.shift + log_scale;
    const double p = exp(lp);
    const double lq = (double(float(x[t.index[first + j]])) - double(st.m)) * inv_t - log_s;
    if (p != 0.0) loss += p * (lp - lq);  // (a slot without mass adds nothing, whatever the student says)
  }
  return float(wave_sum(loss));
}

constexpr int kWaves = kBlock / kWave;

// Maximum and sum of a row, by a whole workgroup.
template <typename T>
__device__ inline SoftmaxSum row_stats(const T *x, uint32_t n, float c, SoftmaxSum *lds) {
  const RowGroups<T> rg(n, 0u);
  SoftmaxSum st = {kMinusInf, 0.0f};
  for (uint32_t g = threadIdx.x; g < rg.groups; g += kBlock) {
    float v[Group<T>::W];
    load_group<T, 0>(rg, x, g, kMinusInf, v);
    fold(st, v, c);
  }
  return block_merge<kWaves>(st, c, lds);
}

// One workgroup a row.
template <typename T>
__global__ __launch_bounds__(kBlock) void distill_kernel(uint32_t n, uint32_t rows, size_t stride, float c, double inv_t,
                                                         const T *__restrict__ x, Teacher t, float *__restrict__ loss,
                                                         float *__restrict__ row_max, float *__restrict__ row_sum) {
  __shared__ SoftmaxSum lds[kWaves];
  for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T *xr = x + r * stride;
    const SoftmaxSum st = row_stats(xr, n, c, lds);
    if (threadIdx.x < uint32_t(kWave)) {
      const float l = row_loss(t, r, xr, n, st, inv_t);
      if (threadIdx.x == 0) {
        loss[r] = l;
        row_max[r] = st.m;
        row_sum[r] = st.s;
      }
    }
  }
}

// The slots of a row while its gradient is written: the classes they name get their value after the dense pass.
struct Slots {
  float *p;         // [k]; 0 for a slot that does not count
  uint32_t *index;  // [k]; kNoClass for a slot that does not count
  float *x;         // [k]: the student's logit, read before dx (which may be x) is written
  float *old;       // [k]: what dx held (accumulating)
};

// dx of one row by a whole workgroup.  dx may be x.
template <typename T, bool ACC>
__device__ inline void row_grad(const T *x, T *dx, uint32_t n, SoftmaxSum st, float c, double inv_t, float dy,
                                const Teacher &t, size_t row, const Slots &slots, double *lds_mass) {
  const size_t first = row * t.k;
  if (threadIdx.x < uint32_t(kWave)) {
    const TeacherRow tr = teacher_row(t, row, n, inv_t);
    for (uint32_t j = threadIdx.x; j < t.k; j += kWave) {
      const bool counts = t.counts(first + j, n);
      const uint32_t at = counts ? t.index[first + j] : kNoClass;
      slots.index[j] = at;
      slots.p[j] = counts ? float(exp(double(t.value[first + j]) * inv_t - tr.shift) * tr.scale) : 0.0f;
      slots.x[j] = counts ? float(x[at]) : 0.0f;
      if (ACC) slots.old[j] = counts ? float(dx[at]) : 0.0f;
    }
    if (threadIdx.x == 0) *lds_mass = tr.any ? tr.mass : -1.0;
  }
  __syncthreads();
  const double mass = *lds_mass;
  const bool any = mass >= 0.0 || mass != mass;  // (a mass that is NaN shows in dx)
  const double w = double(dy) * inv_t;
  const float scale = float(w * mass / double(st.s));
  const RowGroups<T> rg(n, 0u);
  if (any || !ACC) {
    for (uint32_t g = threadIdx.x; g < rg.groups; g += kBlock) {
      float v[Group<T>::W], o[Group<T>::W];
      load_group<T, 0>(rg, x, g, 0.0f, v);
      if (ACC) load_group<T, 0>(rg, dx, g, 0.0f, o);
#pragma unroll
      for (int j = 0; j < Group<T>::W; ++j) {
        v[j] = any ? exp_scaled(v[j], st.m, c) * scale : 0.0f;
        if (ACC) v[j] += o[j];
      }
      if (rg.whole(g)) {
        store_unaligned<int(sizeof(T))>(dx + rg.first(g), pack(v, dx));
      } else {
#pragma unroll
        for (int j = 0; j < Group<T>::W; ++j) {
          if (rg.has(g, j)) dx[size_t(rg.first(g) + uint32_t(j))] = T(v[j]);
        }
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the dense values are written before the slots' values follow
  __syncthreads();
  if (any) {
    for (uint32_t j = threadIdx.x; j < t.k; j += kBlock) {
      const uint32_t at = slots.index[j];
      if (at == kNoClass) continue;
      // slots that name the same class: the first of them writes, with all of their mass, added in slot order
      bool owner = true;
      for (uint32_t i = 0; i < j; ++i) owner &= slots.index[i] != at;
      if (!owner) continue;
      double p = 0.0;
      for (uint32_t i = j; i < t.k; ++i) p += slots.index[i] == at ? double(slots.p[i]) : 0.0;
      const double q = exp((double(slots.x[j]) - double(st.m)) * inv_t) / double(st.s);
      const double g = w * (mass * q - p);
      dx[at] = T(ACC ? float(double(slots.old[j]) + g) : float(g));
    }
  }
  __syncthreads();
}

__device__ inline Slots slots_in(float *lds, uint32_t k) {
  return Slots{lds, reinterpret_cast<uint32_t *>(lds + k), lds + 2u * k, lds + 3u * k};
}

// One workgroup a row.
template <typename T, bool ACC>
__global__ __launch_bounds__(kBlock) void distill_bwd_kernel(uint32_t n, uint32_t rows, size_t stride, float c, double inv_t,
                                                             const float *__restrict__ dy, const T *x, Teacher t,
                                                             const float *__restrict__ row_max,
                                                             const float *__restrict__ row_sum, T *dx) {
  extern __shared__ float slot_lds[];
  __shared__ double mass;
  for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
    row_grad<T, ACC>(x + r * stride, dx + r * stride, n, SoftmaxSum{row_max[r], row_sum[r]}, c, inv_t, dy[r], t, r,
                     slots_in(slot_lds, t.k), &mass);
  }
}

template <typename T>
__global__ __launch_bounds__(kBlock) void distill_fused_kernel(uint32_t n, uint32_t rows, size_t stride, float c,
                                                               double inv_t, const T *x, Teacher t,
                                                               const float *__restrict__ dy, float *__restrict__ loss,
                                                               float *__restrict__ row_max, float *__restrict__ row_sum,
                                                               T *dx) {
  extern __shared__ float slot_lds[];
  __shared__ SoftmaxSum lds[kWaves];
  __shared__ double mass;
  for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T *xr = x + r * stride;
    const SoftmaxSum st = row_stats(xr, n, c, lds);
    if (threadIdx.x < uint32_t(kWave)) {
      const float l = row_loss(t, r, xr, n, st, inv_t);
      if (threadIdx.x == 0) {
        loss[r] = l;
        row_max[r] = st.m;
        row_sum[r] = st.s;
      }
    }
    row_grad<T, false>(xr, dx + r * stride, n, st, c, inv_t, dy[r], t, r, slots_in(slot_lds, t.k), &mass);
  }
}

// ---- host side ----

struct Shape {
  uint32_t n, rows;
  size_t stride;
  float c;
  double inv_t;
};

int prepare(const char *symbol, uint32_t dim0, uint32_t dim1, uint32_t stride, uint32_t k, float temperature, Shape &s) {
  if (const int e = check_rows(symbol, dim0, stride, k, temperature)) return e;
  s = Shape{dim0, dim1, size_t(stride != 0u ? stride : dim0), float(1.4426950408889634 / double(temperature)),
            1.0 / double(temperature)};
  return 0;
}

template <typename T>
int check_arrays(const char *symbol, const Shape &s, const T *x, const Teacher &t, std::initializer_list<const void *> needed) {
  if (s.n != 0u && (x == nullptr || misaligned(x))) return refuse(symbol, "the logits are missing or not aligned to their type");
  if (t.k != 0u && (t.value == nullptr || t.index == nullptr)) return refuse(symbol, "the teacher's slots are missing");
  for (const void *p : needed) {
    if (p == nullptr) return refuse(symbol, "an array is missing");
  }
  return 0;
}

uint32_t row_grid(uint32_t rows) { return rows < (1u << 24) ? rows : (1u << 24); }

template <typename T>
int distill(const char *symbol, uint32_t dim0, uint32_t dim1, uint32_t stride, float temperature, const T *x, const Teacher &t,
            float *loss, float *row_max, float *row_sum, CUstream_st *stream) {
  Shape s;
  if (const int e = prepare(symbol, dim0, dim1, stride, t.k, temperature, s)) return e;
  if (dim1 == 0u) return 0;
  if (const int e = check_arrays(symbol, s, x, t, {loss, row_max, row_sum})) return e;
  distill_kernel<T><<<row_grid(s.rows), kBlock, 0, as_stream(stream)>>>(s.n, s.rows, s.stride, s.c, s.inv_t, x, t, loss,
                                                                        row_max, row_sum);
  note_launch(symbol);
  return 0;
}

template <typename T, bool ACC>
int distill_bwd(const char *symbol, uint32_t dim0, uint32_t dim1, uint32_t stride, float temperature, const float *dy,
                const T *x, const Teacher &t, const float *row_max, const float *row_sum, T *dx, CUstream_st *stream) {
  Shape s;
  if (const int e = prepare(symbol, dim0, dim1, stride, t.k, temperature, s)) return e;
  if (dim1 == 0u || dim0 == 0u) return 0;
  if (const int e = check_arrays(symbol, s, x, t, {dy, row_max, row_sum, dx})) return e;
  if (misaligned(dx)) return refuse(symbol, "the gradient is not aligned to its type");
  distill_bwd_kernel<T, ACC><<<row_grid(s.rows), kBlock, 16u * t.k, as_stream(stream)>>>(
      s.n, s.rows, s.stride, s.c, s.inv_t, dy, x, t, row_max, row_sum, dx);
  note_launch(symbol);
  return 0;
}

template <typename T>
int distill_fused(const char *symbol, uint32_t dim0, uint32_t dim1, uint32_t stride, float temperature, const T *x,
                  const Teacher &t, const float *dy, float *loss, float *row_max, float *row_sum, T *dx, CUstream_st *stream) {
  Shape s;
  if (const int e = prepare(symbol, dim0, dim1, stride, t.k, temperature, s)) return e;
  if (dim1 == 0u) return 0;
  if (const int e = check_arrays(symbol, s, x, t, {dy, loss, row_max, row_sum})) return e;
  if (dim0 != 0u && (dx == nullptr || misaligned(dx))) return refuse(symbol, "the gradient is missing or not aligned to its type");
  distill_fused_kernel<T><<<row_grid(s.rows), kBlock, 16u * t.k, as_stream(stream)>>>(
      s.n, s.rows, s.stride, s.c, s.inv_t, x, t, dy, loss, row_max, row_sum, dx);
  note_launch(symbol);
  return 0;
}

}  // namespace
}  // namespace anode

// One set of entry points for each element type: SUFFIX of the names, ABI type, device type.
#define ANODE_DISTILL(SUFFIX, ABI, DEV)                                                                                       \
  ANODE_EXPORT int anode_gpu_softmax_distill_rows_##SUFFIX(                                                                   \
      uint32_t dim0, uint32_t dim1, uint32_t stride, uint32_t k, float temperature, const ABI *x, const float *teacher_value, \
      const uint32_t *teacher_index, const float *teacher_log_norm, float *loss, float *row_max, float *row_sum,              \
      const KernelConfig *, CUstream_st *stream) {                                                                            \
    return anode::distill<anode::DEV>(__func__, dim0, dim1, stride, temperature, reinterpret_cast<const anode::DEV *>(x),     \
                                      {teacher_value, teacher_index, teacher_log_norm, k}, loss, row_max, row_sum, stream);   \
  }                                                                                                                           \
  ANODE_EXPORT int anode_gpu_softmax_distill_bwd_rows_##SUFFIX(                                                               \
      uint32_t dim0, uint32_t dim1, uint32_t stride, uint32_t k, float temperature, const float *dy, const ABI *x,            \
      const float *teacher_value, const uint32_t *teacher_index, const float *teacher_log_norm, const float *row_max,         \
      const float *row_sum, ABI *dx, const KernelConfig *, CUstream_st *stream) {                                             \
    return anode::distill_bwd<anode::DEV, false>(                                                                             \
        __func__, dim0, dim1, stride, temperature, dy, reinterpret_cast<const anode::DEV *>(x),                               \
        {teacher_value, teacher_index, teacher_log_norm, k}, row_max, row_sum, reinterpret_cast<anode::DEV *>(dx), stream);   \
  }                                                                                                                           \
  ANODE_EXPORT int anode_gpu_softmax_distill_bwd_rows_accumulate_##SUFFIX(                                                    \
      uint32_t dim0, uint32_t dim1, uint32_t stride, uint32_t k, float temperature, const float *dy, const ABI *x,            \
      const float *teacher_value, const uint32_t *teacher_index, const float *teacher_log_norm, const float *row_max,         \
      const float *row_sum, ABI *dx, const KernelConfig *, CUstream_st *stream) {                                             \
    return anode::distill_bwd<anode::DEV, true>(                                                                              \
        __func__, dim0, dim1, stride, temperature, dy, reinterpret_cast<const anode::DEV *>(x),                               \
        {teacher_value, teacher_index, teacher_log_norm, k}, row_max, row_sum, reinterpret_cast<anode::DEV *>(dx), stream);   \
  }                                                                                                                           \
  ANODE_EXPORT int anode_gpu_softmax_distill_fused_fwd_bwd_rows_##SUFFIX(                                                     \
      uint32_t dim0, uint32_t dim1, uint32_t stride, uint32_t k, float temperature, const ABI *x, const float *teacher_value, \
      const uint32_t *teacher_index, const float *teacher_log_norm, const float *dy, float *loss, float *row_max,             \
      float *row_sum, ABI *dx, const KernelConfig *, CUstream_st *stream) {                                                   \
    return anode::distill_fused<anode::DEV>(                                                                                  \
        __func__, dim0, dim1, stride, temperature, reinterpret_cast<const anode::DEV *>(x),                                   \
        {teacher_value, teacher_index, teacher_log_norm, k}, dy, loss, row_max, row_sum,                                      \
        reinterpret_cast<anode::DEV *>(dx), stream);                                                                          \
  }

namespace anode {
typedef float f32_t;
}
ANODE_DISTILL(f32, float, f32_t)
ANODE_DISTILL(bf16, uint16_t, bf16_t)
ANODE_DISTILL(f16, uint16_t, f16_t)
