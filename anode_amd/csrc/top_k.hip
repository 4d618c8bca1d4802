// The k largest values of a row with their classes, and the row's log-sum-exp: what is kept of a teacher's logits for
// distillation (distill.hip), and the candidates for a token.  No kernel of the reference corresponds to it; it
// extends the rule of the arg-max entry points (src/utils/mod.rs:31-41): the larger value first, of equal ones the
// lower class, NaN and -inf never taken.
#include "class_rows.hpp"

namespace anode {
namespace {

constexpr int kTopThreads = 512;
constexpr int kTopWaves = kTopThreads / kWave;

// A value as an unsigned number in the same order, -0 as +0; 0 for what is never taken (NaN, -inf).
__device__ inline uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  const uint32_t key = (b & 0x80000000u) != 0u ? ~b : b | 0x80000000u;
  return (key <= 0x007fffffu || key > 0xff800000u) ? 0u : key;
}
__device__ inline float value_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) != 0u ? key ^ 0x80000000u : ~key);
}

// Leading bits of a key in which two values of the type can differ; the bits below repeat the sign.
template <typename T>
struct KeyBits {
  static constexpr int value = 32;
};
template <>
struct KeyBits<bf16_t> {
  static constexpr int value = 16;
};
template <>
struct KeyBits<f16_t> {
  static constexpr int value = 24;  // sign, eight exponent bits, ten of mantissa; whole digits of 8
};

// An entry: key above, the class inverted below, so that the larger entry comes first in the order of the result.
__device__ inline uint64_t entry_of(uint32_t key, uint32_t k) { return (uint64_t(key) << 32) | uint32_t(~k); }

// Sorts the first `size` (a power of two) entries in LDS, largest first.
template <int THREADS>
__device__ inline void sort_entries(uint64_t *e, uint32_t size) {
  for (uint32_t run = 2; run <= size; run <<= 1) {
    for (uint32_t step = run >> 1; step > 0; step >>= 1) {
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < size / 2; i += THREADS) {
        const uint32_t lo = 2u * i - (i & (step - 1u)), hi = lo + step;
        const uint64_t a = e[lo], b = e[hi];
        if (((lo & run) == 0u) == (a < b)) {
          e[lo] = b;
          e[hi] = a;
        }
      }
    }
  }
  __syncthreads();
}

// One workgroup a row: the k-th largest key is found digit by digit (8 bits a pass over the row, counted in LDS), then
// the larger ones are collected, and of those that equal it the first classes in order; the k entries are sorted.
template <typename T>
__global__ __launch_bounds__(kTopThreads) void top_k_radix_kernel(uint32_t n, uint32_t rows, size_t stride, uint32_t k, Scale sc,
                                                                  double inv_t, const T *__restrict__ x, float *__restrict__ value,
                                                                  uint32_t *__restrict__ index, float *__restrict__ log_norm) {
  constexpr int W = Group<T>::W;
  __shared__ uint64_t entries[kMaxSlots];
  __shared__ uint32_t digits[256];
  __shared__ uint32_t found, above, taken;
  __shared__ uint32_t wave_count[kTopWaves];
  __shared__ SoftmaxSum lds[kTopWaves];
  const uint32_t lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const RowGroups<T> rg(n, 0u);
  for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T *xr = x + r * stride;
    if (log_norm != nullptr) {
      const SoftmaxSum st = finish_stats<T, kTopThreads>(
          stream_stats<T, kTopThreads, 4, 0>(RowSpan<T>(n, 0u), xr, sc), xr, n, sc, lds);
      if (threadIdx.x == 0) log_norm[r] = float(double(st.m) * inv_t + log(double(st.s)));
    }
    uint32_t prefix = 0u, known = 0u, need = k;
    bool all = k == 0u;  // the row holds no more than k values that may be taken (or nothing is asked for)
    for (int shift = 24; shift >= 32 - KeyBits<T>::value && !all; shift -= 8) {
      for (uint32_t i = threadIdx.x; i < 256u; i += kTopThreads) digits[i] = 0u;
      __syncthreads();
      for (uint32_t g = threadIdx.x; g < rg.groups; g += kTopThreads) {
        float v[W];
        load_group<T, 0>(rg, xr, g, kMinusInf, v);
#pragma unroll
        for (int j = 0; j < W; ++j) {
          const uint32_t key = key_of(v[j]);
          if (key != 0u && (key & known) == prefix) atomicAdd(&digits[(key >> shift) & 255u], 1u);
        }
      }
      __syncthreads();
      if (wave == 0) {  // lane l sums the digits 255 - 4 l ... 252 - 4 l, largest first
        uint32_t d[4], own = 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) own += d[i] = digits[255u - 4u * lane - uint32_t(i)];
        uint32_t upto = own;
#pragma unroll
        for (int off = 1; off < kWave; off <<= 1) {
          const uint32_t o = __shfl_up(upto, off, kWave);
          if (int(lane) >= off) upto += o;
        }
        if (lane == 0) found = 256u;
        uint32_t run = upto - own;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (run < need && run + d[i] >= need) {
            found = 255u - 4u * lane - uint32_t(i);
            above = run;
          }
          run += d[i];
        }
      }
      __syncthreads();
      if (found == 256u) {
        all = true;  // (only the first pass can find too few)
      } else {
        need -= above;
        prefix |= found << shift;
        known |= 255u << shift;
      }
      __syncthreads();
    }
    // the k-th largest key; below the digits looked at a key repeats its sign bit, inverted
    uint32_t kth = prefix | ((prefix & 0x80000000u) != 0u ? 0u : ~known);
    if (all) kth = 0u;
    if (threadIdx.x == 0) taken = 0u;
    __syncthreads();
    if (k != 0u) {
      for (uint32_t g = threadIdx.x; g < rg.groups; g += kTopThreads) {
        float v[W];
        load_group<T, 0>(rg, xr, g, kMinusInf, v);
#pragma unroll
        for (int j = 0; j < W; ++j) {
          const uint32_t key = key_of(v[j]);
          if (key > kth) entries[atomicAdd(&taken, 1u)] = entry_of(key, rg.first(g) + uint32_t(j));
        }
      }
    }
    __syncthreads();
    uint32_t count = taken;
    if (!all) {
      // the first `need` classes whose key is the k-th: a workgroup's groups in turn, counted across its threads
      uint32_t before = 0u;
      for (uint32_t base = 0; base < rg.groups && before < need; base += kTopThreads) {
        const uint32_t g = base + threadIdx.x;
        uint32_t same = 0u;
        if (g < rg.groups) {
          float v[W];
          load_group<T, 0>(rg, xr, g, kMinusInf, v);
#pragma unroll
          for (int j = 0; j < W; ++j) same |= uint32_t(key_of(v[j]) == kth) << j;
        }
        const uint32_t own = uint32_t(__popc(same));
        uint32_t upto = own;
#pragma unroll
        for (int off = 1; off < kWave; off <<= 1) {
          const uint32_t o = __shfl_up(upto, off, kWave);
          if (int(lane) >= off) upto += o;
        }
        if (lane == kWave - 1) wave_count[wave] = upto;
        __syncthreads();
        uint32_t at = before + upto - own, total = 0u;
#pragma unroll
        for (int w = 0; w < kTopWaves; ++w) {
          if (uint32_t(w) < wave) at += wave_count[w];
          total += wave_count[w];
        }
        while (same != 0u && at < need) {
          const uint32_t j = uint32_t(__ffs(int(same))) - 1u;
          same &= same - 1u;
          entries[count + at++] = entry_of(kth, rg.first(g) + j);
        }
        before += total;
        __syncthreads();
      }
      count += need;
    }
    uint32_t size = 2u;
    while (size < count) size <<= 1;
    for (uint32_t i = count + threadIdx.x; i < size; i += kTopThreads) entries[i] = 0u;
    sort_entries<kTopThreads>(entries, size);
    for (uint32_t i = threadIdx.x; i < k; i += kTopThreads) {
      const bool have = i < count;
      value[r * k + i] = have ? value_of(uint32_t(entries[i] >> 32)) : kMinusInf;
      index[r * k + i] = have ? ~uint32_t(entries[i]) : kNoClass;
    }
    __syncthreads();
  }
}

template <typename T>
int top_k(const char *symbol, uint32_t dim0, uint32_t dim1, uint32_t stride, uint32_t k, float temperature, const T *x,
          float *value, uint32_t *index, float *log_norm, CUstream_st *stream) {
  if (const int e = check_rows(symbol, dim0, stride, k, temperature)) return e;
  if (dim1 == 0u || (k == 0u && log_norm == nullptr)) return 0;
  if (dim0 != 0u && (x == nullptr || misaligned(x))) return refuse(symbol, "the logits are missing or not aligned to their type");
  if (k != 0u && (value == nullptr || index == nullptr)) return refuse(symbol, "an array is missing");
  const uint32_t grid = dim1 < (1u << 24) ? dim1 : (1u << 24);
  top_k_radix_kernel<T><<<grid, kTopThreads, 0, as_stream(stream)>>>(
      dim0, dim1, size_t(stride != 0u ? stride : dim0), k, scale_for(temperature), 1.0 / double(temperature), x, value, index, log_norm);
  note_launch(symbol);
  return 0;
}

}  // namespace
}  // namespace anode

ANODE_EXPORT int anode_gpu_top_k_rows_f32(uint32_t dim0, uint32_t dim1, uint32_t stride, uint32_t k, float temperature,
                                          const float *x, float *value, uint32_t *index, float *log_norm,
                                          const KernelConfig *, CUstream_st *stream) {
  return anode::top_k(__func__, dim0, dim1, stride, k, temperature, x, value, index, log_norm, stream);
}

ANODE_EXPORT int anode_gpu_top_k_rows_bf16(uint32_t dim0, uint32_t dim1, uint32_t stride, uint32_t k, float temperature,
                                           const uint16_t *x, float *value, uint32_t *index, float *log_norm,
                                           const KernelConfig *, CUstream_st *stream) {
  return anode::top_k(__func__, dim0, dim1, stride, k, temperature, reinterpret_cast<const anode::bf16_t *>(x), value, index,
                      log_norm, stream);
}

ANODE_EXPORT int anode_gpu_top_k_rows_f16(uint32_t dim0, uint32_t dim1, uint32_t stride, uint32_t k, float temperature,
                                          const uint16_t *x, float *value, uint32_t *index, float *log_norm,
                                          const KernelConfig *, CUstream_st *stream) {
  return anode::top_k(__func__, dim0, dim1, stride, k, temperature, reinterpret_cast<const anode::f16_t *>(x), value, index,
                      log_norm, stream);
}
