// The k largest values of a row with their classes, and the row's log-sum-exp: what is kept of a teacher's logits for
// distillation (distill.hip), and the candidates for a token.  No kernel of the reference corresponds to it; it
// extends the rule of the arg-max entry points (src/utils/mod.rs:31-41): the larger value first, of equal ones the
// lower class, NaN and -inf never taken.
#include "class_rows.hpp"

namespace anode {
namespace {

// A value as an unsigned number in the same order, -0 as +0; 0 for what is never taken (NaN, -inf).
constexpr uint32_t kLowestKey = 0x00800000u;  // the lowest finite value's
__device__ inline uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  const uint32_t key = (b & 0x80000000u) != 0u ? ~b : b | 0x80000000u;
  return (key < kLowestKey || key > 0xff800000u) ? 0u : key;
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
// Entries of a row are all different.
__device__ inline uint64_t entry_of(uint32_t key, uint32_t k) { return (uint64_t(key) << 32) | uint32_t(~k); }
__device__ inline uint32_t key_in(uint64_t entry) { return uint32_t(entry >> 32); }

// Sorts the first `size` (a power of two) entries in LDS, largest first.
template <int THREADS>
__device__ inline void sort_entries(uint64_t *e, uint32_t size) {
  for (uint32_t run = 2; run <= size; run <<= 1) {
    for (uint32_t step = run >> 1; step > 0; step >>= 1) {
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < size / 2u; i += THREADS) {
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

// A key that at least j lanes reach, found bit by bit: its leading 18 bits for floats (those below are 0), exactly for the
// 16-bit types, whose keys have no more; 0 where fewer lanes hold a key at all.  The comparisons' results are scalar, so a
// step is a compare, a count and a select.
template <typename T>
__device__ inline uint32_t key_reached_by(uint32_t key, uint32_t j) {
  constexpr int kLow = sizeof(T) == 4 ? 14 : KeyBits<T>::value == 16 ? 16 : 13;
  uint32_t t = 0u;
#pragma unroll
  for (int bit = 31; bit >= kLow; --bit) {
    const uint32_t higher = t | (1u << bit);
    if (uint32_t(__popcll(__ballot(key >= higher))) >= j) t = higher;
  }
  if (sizeof(T) == 2 && t != 0u && (t & 0x80000000u) == 0u) t |= (1u << kLow) - 1u;  // (below its bits a key repeats its sign, inverted)
  return t;
}

// What the exact selection of k entries needs in LDS.
struct RadixLds {
  uint32_t digits[256];
  uint32_t wave_count[16];
  uint32_t found, above, taken;
};

// The entries of a row whose key is above `border`, unsorted into `entries` (room for `most`, k at least): all of them where they
// are k or more, else with the first classes in order of those that equal the border, k together (fewer where the row
// has fewer).  Returns their number, kNoClass where there is no room.
template <typename T, int THREADS>
__device__ inline uint32_t collect(const T *xr, uint32_t n, uint32_t from, uint32_t border, uint32_t k, uint64_t *entries,
                                   uint32_t most, RadixLds &l) {
  constexpr int W = Group<T>::W;
  constexpr int WAVES = THREADS / kWave;
  const uint32_t lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const RowGroups<T> rg(n);
  __syncthreads();
  if (threadIdx.x == 0) l.taken = 0u;
  __syncthreads();
  for (uint32_t g = threadIdx.x; g < rg.groups; g += THREADS) {
    float v[W];
    load_group<T>(rg, xr, g, kMinusInf, v);
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const uint32_t key = key_of(v[j]);
      if (key > border) {
        const uint32_t at = atomicAdd(&l.taken, 1u);
        if (at < most) entries[at] = entry_of(key, from + rg.first(g) + uint32_t(j));
      }
    }
  }
  __syncthreads();
  const uint32_t count = l.taken;
  if (count > most) return kNoClass;
  if (count >= k || border == 0u) return count;
  // the workgroup's groups in turn, counted across its threads
  const uint32_t need = k - count;
  uint32_t before = 0u;
  for (uint32_t base = 0; base < rg.groups && before < need; base += THREADS) {
    const uint32_t g = base + threadIdx.x;
    uint32_t same = 0u;
    if (g < rg.groups) {
      float v[W];
      load_group<T>(rg, xr, g, kMinusInf, v);
#pragma unroll
      for (int j = 0; j < W; ++j) same |= uint32_t(key_of(v[j]) == border) << j;
    }
    const uint32_t own = uint32_t(__popc(same));
    const uint32_t upto = lanes_upto(own);
    if (lane == kWave - 1) l.wave_count[wave] = upto;
    __syncthreads();
    uint32_t at = before + upto - own, total = 0u;
    for (int w = 0; w < WAVES; ++w) {
      if (uint32_t(w) < wave) at += l.wave_count[w];
      total += l.wave_count[w];
    }
    while (same != 0u && at < need) {
      const uint32_t j = uint32_t(__ffs(int(same))) - 1u;
      same &= same - 1u;
      entries[count + at++] = entry_of(border, from + rg.first(g) + j);
    }
    before += total;
    __syncthreads();
  }
  return count + min(need, before);
}

// The k largest entries of a row, or all of them where there are fewer, unsorted into `entries`; returns how many.  Exact
// whatever the row holds: the k-th largest key is found digit by digit (8 bits a pass over the row, counted in LDS; a wave whose
// digits are all alike, as in a row of ties, counts them with one addition), then collect().
template <typename T, int THREADS>
__device__ inline uint32_t radix_select(const T *xr, uint32_t n, uint32_t from, uint32_t k, uint64_t *entries, RadixLds &l) {
  constexpr int W = Group<T>::W;
  const uint32_t lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const RowGroups<T> rg(n);
  uint32_t prefix = 0u, known = 0u, need = k;
  bool all = false;  // the row holds fewer than k values that may be taken
  for (int shift = 24; shift >= 32 - KeyBits<T>::value && !all; shift -= 8) {
    for (uint32_t i = threadIdx.x; i < 256u; i += THREADS) l.digits[i] = 0u;
    __syncthreads();
    for (uint32_t g = threadIdx.x; g < rg.groups; g += THREADS) {
      float v[W];
      load_group<T>(rg, xr, g, kMinusInf, v);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const uint32_t key = key_of(v[j]), digit = (key >> shift) & 255u;
        if (key != 0u && (key & known) == prefix) {
          const uint64_t here = __ballot(true);
          if (__all(digit == uint32_t(__builtin_amdgcn_readfirstlane(int(digit))))) {
            if (lane == uint32_t(__ffsll((unsigned long long)here)) - 1u) atomicAdd(&l.digits[digit], uint32_t(__popcll(here)));
          } else {
            atomicAdd(&l.digits[digit], 1u);
          }
        }
      }
    }
    __syncthreads();
    if (wave == 0) {  // lane i sums the digits 255 - 4 i ... 252 - 4 i, largest first
      uint32_t d[4], own = 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) own += d[i] = l.digits[255u - 4u * lane - uint32_t(i)];
      uint32_t run = lanes_upto(own) - own;
      if (lane == 0) l.found = 256u;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (run < need && run + d[i] >= need) {
          l.found = 255u - 4u * lane - uint32_t(i);
          l.above = run;
        }
        run += d[i];
      }
    }
    __syncthreads();
    if (l.found == 256u) {
      all = true;  // (only the first pass can find too few)
    } else {
      need -= l.above;
      prefix |= l.found << shift;
      known |= 255u << shift;
    }
    __syncthreads();
  }
  // the k-th largest key; below the digits looked at a key repeats its sign bit, inverted
  const uint32_t kth = all ? 0u : prefix | ((prefix & 0x80000000u) != 0u ? 0u : ~known);
  return collect<T, THREADS>(xr, n, from, kth, k, entries, k, l);
}

// The entries in LDS that can be among the k largest, to `out` (room for `most`): those that reach a key which k of them
// reach, and few more.  Returns their number, which may be above `most` (then `out` is incomplete).
template <typename T, int THREADS>
__device__ inline uint32_t drop_small(const uint64_t *entries, uint32_t count, uint32_t k, uint64_t *out, uint32_t most,
                                      uint32_t *wave_key, uint32_t *taken) {
  constexpr uint32_t WAVES = THREADS / kWave;
  uint32_t top = 0u;
  for (uint32_t i = threadIdx.x; i < count; i += THREADS) top = max(top, key_in(entries[i]));
  const uint32_t t = key_reached_by<T>(top, (k + WAVES - 1u) / WAVES);
  if ((threadIdx.x & (kWave - 1)) == 0) wave_key[threadIdx.x / kWave] = t;
  if (threadIdx.x == 0) *taken = 0u;
  __syncthreads();
  uint32_t least = wave_key[0];
#pragma unroll
  for (uint32_t w = 1; w < WAVES; ++w) least = min(least, wave_key[w]);
  for (uint32_t i = threadIdx.x; i < count; i += THREADS) {
    const uint64_t e = entries[i];
    if (key_in(e) >= least) {
      const uint32_t at = atomicAdd(taken, 1u);
      if (at < most) out[at] = e;
    }
  }
  __syncthreads();
  return *taken;
}

// The selection where the list was too short, out of line: inlined it costs the streaming loop registers (119 against 114 us).  With
// the threshold that the whole row gives -- `top` is the thread's largest value -- it reads the row once more; that settles
// rising rows, and ties at the threshold itself (zeros, a mask's lowest value), of which the first in order are
// wanted.  Else the exact k-th key is found.  The result is in `best`.
template <typename T, int THREADS>
__device__ __attribute__((noinline)) uint32_t select_again(const T *xr, uint32_t n, uint32_t from, float top, uint32_t k, uint64_t *list,
                                                           uint32_t room, uint64_t *best, uint32_t most, RadixLds *l) {
  constexpr uint32_t WAVES = THREADS / kWave;
  const uint32_t t = key_reached_by<T>(key_of(top), (k + WAVES - 1u) / WAVES);
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) l->wave_count[threadIdx.x / kWave] = t;
  __syncthreads();
  uint32_t border = l->wave_count[0];
  for (uint32_t w = 1; w < WAVES; ++w) border = min(border, l->wave_count[w]);
  uint32_t have = collect<T, THREADS>(xr, n, from, border, k, list, room, *l);
  __syncthreads();
  if (have != kNoClass) {
    have = drop_small<T, THREADS>(list, have, k, best, most, l->wave_count, &l->taken);
    if (have <= most) return have;
  }
  __syncthreads();
  have = radix_select<T, THREADS>(xr, n, from, k, best, *l);
  __syncthreads();
  return have;
}

// The result of a row from its entries in LDS, at least the k largest of them, and empty slots behind.  Up to 256 entries are
// counted against each other (a thread an entry, the others read two at a time by all lanes alike); more are sorted.
template <int THREADS>
__device__ inline void write_result(uint64_t *entries, uint32_t count, size_t row, uint32_t k, float *value, uint32_t *index) {
  if (count <= 256u) {
    if (threadIdx.x == 0u) entries[count] = 0u;  // (the second of the last pair; the array has room)
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < count; i += THREADS) {
      const uint64_t own = entries[i];
      uint32_t rank = 0u;
      for (uint32_t j = 0; j < count; j += 2) {
        typedef uint64_t pair __attribute__((ext_vector_type(2)));
        const pair e = *reinterpret_cast<const pair *>(&entries[j]);
        rank += (e.x > own ? 1u : 0u) + (e.y > own ? 1u : 0u);
      }
      if (rank < k) {
        value[row * k + rank] = value_of(key_in(own));
        index[row * k + rank] = ~uint32_t(own);
      }
    }
  } else {
    uint32_t size = 2u;
    while (size < count) size <<= 1;
    for (uint32_t i = count + threadIdx.x; i < size; i += THREADS) entries[i] = 0u;
    sort_entries<THREADS>(entries, size);
    for (uint32_t i = threadIdx.x; i < k && i < count; i += THREADS) {
      value[row * k + i] = value_of(key_in(entries[i]));
      index[row * k + i] = ~uint32_t(entries[i]);
    }
  }
  for (uint32_t i = count + threadIdx.x; i < k; i += THREADS) {
    value[row * k + i] = kMinusInf;
    index[row * k + i] = kNoClass;
  }
}

// A part of a row: rows are cut into `parts` of `per` values where there are too few to fill the GPU.
struct Cut {
  uint32_t parts, per;
};

// What the parts of a row leave for the kernel that joins them.
struct PartResults {
  uint64_t *entries;  // [quota, parts, rows]
  uint32_t *count;    // [parts, rows]
  SoftmaxSum *stats;  // [parts, rows]
  uint32_t quota;
};

// One workgroup a part of a row, which it reads once.  A threshold that k values seen so far reach -- every wave finds what its
// share of k reaches among the largest value of each of its lanes, the least of the waves counts -- is renewed after 1, 2, 4,
// 8 ... tiles; values that reach it are put into a list in LDS, which grows by little more than k between two renewals, whatever
// the row's length.  What the list holds at the end is thinned the same way, sorted and written.  Rows for which the list
// is too short (thousands of ties at the threshold, the largest values all in few lanes' places, rising rows) are read again.
template <typename T, int THREADS, int LIST, bool NORM>
__global__ __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(THREADS > 512 ? 8 : THREADS > 256 ? 6 : 5))) void top_k_kernel(
    uint32_t n, uint32_t rows, size_t stride, uint32_t k, Scale sc, double inv_t, Cut cut, const T *__restrict__ x,
    float *__restrict__ value, uint32_t *__restrict__ index, float *__restrict__ log_norm, PartResults pr) {
  constexpr int W = Group<T>::W;
  constexpr int U = THREADS > 256 ? 16 / W : 4;  // groups of a thread together
  constexpr uint32_t WAVES = THREADS / kWave;
  constexpr uint32_t kTile = uint32_t(THREADS) * uint32_t(U);
  constexpr uint32_t kShort = THREADS > 256 ? 2u * uint32_t(THREADS) : 512u;
  __shared__ __align__(16) uint64_t list[LIST];
  __shared__ __align__(16) uint64_t best[kShort];
  __shared__ RadixLds radix;
  __shared__ uint32_t wave_key[2][WAVES];
  __shared__ uint32_t listed, taken;
  __shared__ SoftmaxSum sums[WAVES];
  const uint32_t wave = threadIdx.x / kWave;
  const uint32_t share = (k + WAVES - 1u) / WAVES;
  const uint64_t items = uint64_t(rows) * cut.parts;
  for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const size_t r = item / cut.parts;
    const uint32_t from = uint32_t(item % cut.parts) * cut.per;
    const uint32_t count = min(cut.per, n - from);
    const T *xr = x + r * stride + from;
    const RowSpan<T> span(count, 0u);
    if (threadIdx.x == 0) listed = 0u;
    __syncthreads();
    float top = kMinusInf, least = -__FLT_MAX__;
    SoftmaxSum st = {-sc.limit, 0.0f};
    bool full = false;  // this thread has seen the list overflow
    auto put = [&](float v, uint32_t at) {
      if (v >= least) {
        const uint32_t place = atomicAdd(&listed, 1u);
        if (place < uint32_t(LIST)) {
          list[place] = entry_of(key_of(v), from + at);
        } else {
          full = true;
        }
      }
    };
    if (span.groups != 0u) {
      u32x4 q[U];
      load_tile<T, THREADS, U>(span, xr, threadIdx.x, q);
      uint32_t tile = 0u, turn = 0u;
      for (uint32_t base = 0;; base += kTile, ++tile) {
        float v[U * W];
        u32x4 next[U];
        const bool more = span.groups - base > kTile;
        load_tile<T, THREADS, U>(span, xr, base + kTile + threadIdx.x, next);
        unpack_tile<T, U>(q, v);
        if (!more) mask_tile<T, THREADS, U>(span, base + threadIdx.x, kMinusInf, v);
        const float tile_top = max_of(kMinusInf, v);
        top = fmaxf(top, tile_top);
        if ((tile & (tile - 1u)) == 0u) {
          const uint32_t t = key_reached_by<T>(key_of(top), share);
          uint32_t *keys = wave_key[turn];  // (the other half may still be read)
          turn ^= 1u;
          if ((threadIdx.x & (kWave - 1)) == 0) keys[wave] = t;
          __syncthreads();
          uint32_t low = keys[0];
#pragma unroll
          for (uint32_t w = 1; w < WAVES; ++w) low = min(low, keys[w]);
          least = low < kLowestKey ? -__FLT_MAX__ : value_of(low);
        }
        if (tile_top >= least && !full) {  // (rare: the values are marked and fetched again; an indexed register is dearer)
          uint32_t marked = 0u;
#pragma unroll
          for (int i = 0; i < U * W; ++i) marked |= uint32_t(v[i] >= least) << i;
          do {
            const uint32_t i = uint32_t(__ffs(int(marked))) - 1u;
            marked &= marked - 1u;
            const uint32_t at = span.first(base + threadIdx.x + i / uint32_t(W) * uint32_t(THREADS)) + i % uint32_t(W);
            put(float(xr[at]), at);
          } while (marked != 0u);
        }
        if constexpr (NORM) fold_below(st, fmaxf(top, -sc.limit), v, sc.c);
        if (!more) break;
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = next[u];
      }
    }
    if (span.single(threadIdx.x)) {  // (at most 7: the head is empty)
      const uint32_t at = span.single_at(threadIdx.x);
      const float v = float(xr[at]);
      put(v, at);
      if constexpr (NORM) fold_one(st, v, sc.c);
    }
    __syncthreads();
    uint32_t have = listed;
    if (have <= uint32_t(LIST)) have = drop_small<T, THREADS>(list, have, k, best, kShort, wave_key[0], &taken);
    if (have > kShort) have = select_again<T, THREADS>(xr, count, from, top, k, list, uint32_t(LIST), best, kShort, &radix);
    if (cut.parts > 1u && have > pr.quota) {  // more than the part has room for: the k largest of them
      uint32_t size = 2u;
      while (size < have) size <<= 1;
      for (uint32_t i = have + threadIdx.x; i < size; i += THREADS) best[i] = 0u;
      sort_entries<THREADS>(best, size);
      have = k;
    }
    if (cut.parts == 1u) {
      write_result<THREADS>(best, have, r, k, value, index);
      if constexpr (NORM) {
        st = finish_stats<T, THREADS>(st, xr, n, sc, sums);
        if (threadIdx.x == 0) log_norm[r] = float(double(st.m) * inv_t + log(double(st.s)));
      }
    } else {
      for (uint32_t i = threadIdx.x; i < have; i += THREADS) pr.entries[item * pr.quota + i] = best[i];
      if (threadIdx.x == 0) pr.count[item] = have;
      if constexpr (NORM) {
        st = block_merge<WAVES>(st, sc.c, sums);
        if (threadIdx.x == 0) pr.stats[item] = st;
      }
    }
    __syncthreads();
  }
}

// One workgroup a row: its parts' entries together, thinned, sorted and written.
constexpr uint32_t kJoined = 4096;  // entries of a row's parts at most
template <typename T, bool NORM>
__global__ __launch_bounds__(kBlock) void top_k_join_kernel(uint32_t n, uint32_t rows, size_t stride, uint32_t k, Scale sc,
                                                            double inv_t, uint32_t parts, const T *__restrict__ x,
                                                            float *__restrict__ value, uint32_t *__restrict__ index,
                                                            float *__restrict__ log_norm, PartResults pr) {
  constexpr uint32_t kShort = 2048;
  __shared__ __align__(16) uint64_t list[kJoined];
  __shared__ __align__(16) uint64_t best[kShort];
  __shared__ uint32_t first[65];
  __shared__ uint32_t wave_key[kBlock / kWave];
  __shared__ uint32_t taken;
  __shared__ float plain_lds[kBlock / kWave];
  for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
    SoftmaxSum st = {-sc.limit, 0.0f};
    if constexpr (NORM) {
      const uint32_t lane = threadIdx.x & (kWave - 1);
      if (lane < parts) st = pr.stats[r * parts + lane];
    }
    // (at most 64 parts: a lane finds where its part's entries begin, a thread which part its entry is of)
    if (threadIdx.x < uint32_t(kWave)) {
      const uint32_t count = threadIdx.x < parts ? pr.count[r * parts + threadIdx.x] : 0u;
      first[threadIdx.x + 1u] = lanes_upto(count);
      if (threadIdx.x == 0u) first[0] = 0u;
    }
    __syncthreads();
    const uint32_t have = first[kWave];
    for (uint32_t i = threadIdx.x; i < have; i += kBlock) {
      uint32_t part = 0u;
#pragma unroll
      for (uint32_t step = 32u; step > 0u; step >>= 1) part += first[part + step] <= i ? step : 0u;
      list[i] = pr.entries[(r * parts + part) * pr.quota + (i - first[part])];
    }
    __syncthreads();
    const uint32_t few = drop_small<T, kBlock>(list, have, k, best, kShort, wave_key, &taken);
    if (few <= kShort) {
      write_result<kBlock>(best, few, r, k, value, index);
    } else {
      write_result<kBlock>(list, have, r, k, value, index);
    }
    if constexpr (NORM) {
      st = wave_merge(st, sc.c);
      if (measured(st.m, sc)) {
        st.s = true_sum(st, sc.c);
      } else {
        st = plain_stats<T, kBlock>(x + r * stride, n, sc.c, plain_lds);
      }
      if (threadIdx.x == 0) log_norm[r] = float(double(st.m) * inv_t + log(double(st.s)));
    }
    __syncthreads();
  }
}

// Threads of a workgroup: a wave's 64 lanes speak for its share of k, so two or four waves take up to 128, eight up to 256, sixteen
// more.  Two for short rows: 65536 rows of 1000 floats 100 against 200 us, 8192 of 16000 bf16 62 against 74; 1024 of 32768
// 35 against 28.  Eight for k = 200: 156 against 203 us with sixteen.
uint32_t threads_for(uint32_t n, uint32_t k) { return k > 256u ? 1024u : k > 128u ? 512u : n <= 16384u ? 128u : 256u; }

// Parts of at least 4096 values, no more than bring the launch to eight waves a CU, and with room for three times k entries
// each among those that are joined (a part leaves little more than k).
Cut cut_row(uint32_t n, uint32_t rows, uint32_t k, uint32_t threads) {
  uint64_t parts = uint64_t(device_cu_count()) * (512u / threads) / rows;
  if (parts > n / 4096u) parts = n / 4096u;
  if (parts > 64u) parts = 64u;
  if (k != 0u && parts > kJoined / (3u * k)) parts = kJoined / (3u * k);
  if (parts <= 1u) return Cut{1u, n};
  const uint64_t per = ((uint64_t(n) + parts - 1u) / parts + 1023u) / 1024u * 1024u;
  return Cut{uint32_t((n + per - 1u) / per), uint32_t(per)};
}
struct PartBytes {
  size_t entries, stats, counts;
};
PartBytes part_bytes(uint32_t rows, const Cut &cut) {
  const size_t items = size_t(rows) * cut.parts;
  return PartBytes{items * (kJoined / cut.parts) * sizeof(uint64_t), items * sizeof(SoftmaxSum), items * sizeof(uint32_t)};
}

template <typename T, int THREADS, int LIST, bool NORM>
int launch_top_k(const char *symbol, uint32_t n, uint32_t rows, size_t stride, uint32_t k, float temperature, const T *x,
                 float *value, uint32_t *index, float *log_norm, hipStream_t st) {
  const Cut cut = cut_row(n, rows, k, THREADS);
  const uint64_t items = uint64_t(rows) * cut.parts;
  const uint32_t most = 1u << 24, grid = items < most ? uint32_t(items) : most;
  const Scale sc = scale_for(temperature);
  const double inv_t = 1.0 / double(temperature);
  PartResults pr = {nullptr, nullptr, nullptr, kJoined / cut.parts};
  if (cut.parts == 1u) {
    top_k_kernel<T, THREADS, LIST, NORM><<<grid, THREADS, 0, st>>>(n, rows, stride, k, sc, inv_t, cut, x, value, index, log_norm, pr);
  } else {
    const PartBytes bytes = part_bytes(rows, cut);
    const RowsScratch scratch = rows_scratch(st, bytes.entries + bytes.stats + bytes.counts, symbol);
    if (scratch.error != 0) return scratch.error;
    char *at = static_cast<char *>(scratch.lease.ptr);
    pr.entries = reinterpret_cast<uint64_t *>(at);
    pr.stats = reinterpret_cast<SoftmaxSum *>(at + bytes.entries);
    pr.count = reinterpret_cast<uint32_t *>(at + bytes.entries + bytes.stats);
    top_k_kernel<T, THREADS, LIST, NORM><<<grid, THREADS, 0, st>>>(n, rows, stride, k, sc, inv_t, cut, x, value, index, log_norm, pr);
    top_k_join_kernel<T, NORM><<<rows < most ? rows : most, kBlock, 0, st>>>(n, rows, stride, k, sc, inv_t, cut.parts, x, value,
                                                                           index, log_norm, pr);
  }
  note_launch(symbol);
  return 0;
}

template <typename T>
int top_k(const char *symbol, uint32_t dim0, uint32_t dim1, uint32_t stride, uint32_t k, float temperature, const T *x,
          float *value, uint32_t *index, float *log_norm, CUstream_st *stream) {
  if (const int e = check_rows(symbol, dim0, stride, k, temperature)) return e;
  if (dim1 == 0u || (k == 0u && log_norm == nullptr)) return 0;
  if (dim0 != 0u && (x == nullptr || misaligned(x))) return refuse(symbol, "the logits are missing or not aligned to their type");
  if (k != 0u && (value == nullptr || index == nullptr)) return refuse(symbol, "an array is missing");
  const size_t pitch = stride != 0u ? stride : dim0;
  const hipStream_t st = as_stream(stream);
  auto go = [&](auto norm) {
    constexpr bool NORM = decltype(norm)::value;
    switch (threads_for(dim0, k)) {
      case 128u: return launch_top_k<T, 128, 1024, NORM>(symbol, dim0, dim1, pitch, k, temperature, x, value, index, log_norm, st);
      case 256u: return launch_top_k<T, 256, 1536, NORM>(symbol, dim0, dim1, pitch, k, temperature, x, value, index, log_norm, st);
      case 512u: return launch_top_k<T, 512, 2560, NORM>(symbol, dim0, dim1, pitch, k, temperature, x, value, index, log_norm, st);
      default: return launch_top_k<T, 1024, 4096, NORM>(symbol, dim0, dim1, pitch, k, temperature, x, value, index, log_norm, st);
    }
  };
  return log_norm != nullptr ? go(std::true_type{}) : go(std::false_type{});
}

}  // namespace

size_t top_k_scratch(uint32_t classes, uint32_t rows, uint32_t k) {
  if (rows == 0u || k > kMaxSlots) return 0u;
  const Cut cut = cut_row(classes, rows, k, threads_for(classes, k));
  if (cut.parts == 1u) return 0u;
  const PartBytes b = part_bytes(rows, cut);
  return b.entries + b.stats + b.counts;
}
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
