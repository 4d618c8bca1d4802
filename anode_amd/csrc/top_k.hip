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

// The lowest bit of a key that the searches below look at: 18 leading bits of floats (those below are 0), all of the 16-bit
// types', whose keys have no more.
template <typename T>
struct LowestBit {
  static constexpr uint32_t value = sizeof(T) == 4 ? 1u << 14 : KeyBits<T>::value == 16 ? 1u << 16 : 1u << 13;
};
template <typename T>
__device__ inline uint32_t whole_key(uint32_t t) {  // (below its bits a key of a 16-bit type repeats its sign, inverted)
  return sizeof(T) == 2 && t != 0u && (t & 0x80000000u) == 0u ? t | (LowestBit<T>::value - 1u) : t;
}

// A key that at least j lanes reach, found bit by bit; 0 where fewer lanes hold a key at all.  The comparisons' results are
// scalar, so a step is a compare, a count and a select.
template <typename T>
__device__ inline uint32_t key_reached_by(uint32_t key, uint32_t j) {
  uint32_t t = 0u;
#pragma unroll
  for (uint32_t bit = 0x80000000u; bit >= LowestBit<T>::value; bit >>= 1) {
    if (uint32_t(__popcll(__ballot(key >= (t | bit)))) >= j) t |= bit;
  }
  return whole_key<T>(t);
}

constexpr int kSegments = 16;  // of a thread, whose largest values lie in LDS

// Room for `own` items of this lane behind a counter in LDS; the wave's lanes all call it.  (One addition for the wave: given an
// atomic addition of different amounts the compiler adds the lanes up one after the other, 2 us of a row.)
__device__ inline uint32_t reserve(uint32_t *counter, uint32_t own) {
  const uint32_t upto = lanes_upto(own), all = from_lane(upto, kWave - 1);
  uint32_t at = 0u;
  if (all != 0u) {
    if ((threadIdx.x & (kWave - 1)) == 0u) at = atomicAdd(counter, all);
    at = from_lane(at, 0);
  }
  return at + upto - own;
}

// What the exact selection of k entries needs in LDS.
struct RadixLds {
  uint32_t digits[256];
  uint32_t wave_count[16];  // (two for each of eight waves)
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

constexpr uint32_t kCounted = 256;  // entries that are ranked by counting, at most

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

// The same, of at most MOST entries, by the k-th largest key itself but for its low bits: no more than k and those that equal it.
// A thread holds its share of the entries in registers; the key is found bit by bit, the waves' counts meet in LDS.  (Out of line: few rows need it.)
template <typename T, int THREADS, int MOST>
__device__ __attribute__((noinline)) uint32_t drop_all_but(const uint64_t *entries, uint32_t count, uint32_t k, uint64_t *out, uint32_t most,
                                      uint32_t *wave_count, uint32_t *taken) {
  constexpr uint32_t WAVES = THREADS / kWave;
  constexpr int EACH = MOST / THREADS;
  static_assert(MOST % THREADS == 0, "a thread's share");
  const uint32_t wave = threadIdx.x / kWave;
  uint64_t own[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const uint32_t i = threadIdx.x + uint32_t(e * THREADS);
    own[e] = i < count ? entries[i] : 0u;
  }
  if (threadIdx.x == 0) *taken = 0u;
  uint32_t least = 0u, turn = 0u;
#pragma unroll 1
  for (uint32_t bit = 0x80000000u; bit >= LowestBit<T>::value; bit >>= 1) {
    uint32_t reached = 0u;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      if (uint32_t(e * THREADS) < count) reached += uint32_t(__popcll(__ballot(key_in(own[e]) >= (least | bit))));
    }
    if constexpr (WAVES > 1) {
      // (two halves in turn, so that one barrier a bit is enough)
      if ((threadIdx.x & (kWave - 1)) == 0) wave_count[turn + wave] = reached;
      __syncthreads();
      reached = 0u;
#pragma unroll
      for (uint32_t w = 0; w < WAVES; ++w) reached += wave_count[turn + w];
      turn ^= WAVES;
    }
    if (reached >= k) least |= bit;
  }
  least = whole_key<T>(least);
  __syncthreads();
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    if (uint32_t(e * THREADS) >= count) break;
    const bool in = key_in(own[e]) != 0u && key_in(own[e]) >= least;
    const uint32_t at = reserve(taken, in ? 1u : 0u);
    if (in && at < most) out[at] = own[e];
  }
  __syncthreads();
  return *taken;
}

// Entries thinned until they fit in `out`, the quick way first: 8 rows of 1024 halves, of which 165 are kept, 22 against 37 us that
// sorting all of them takes.  (Where the quick way is enough it is the quicker: 8192 rows of 16000 bf16, k = 200, 109
// against 116 us.)
template <typename T, int THREADS, int MOST>
__device__ inline uint32_t thin_out(const uint64_t *entries, uint32_t count, uint32_t k, uint64_t *out, uint32_t most, uint32_t *waves,
                                    uint32_t *taken) {
  const uint32_t few = drop_small<T, THREADS>(entries, count, k, out, most, waves, taken);
  if (few <= most) return few;
  __syncthreads();
  return drop_all_but<T, THREADS, MOST>(entries, count, k, out, most, waves, taken);
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
    have = thin_out<T, THREADS, kSegments * THREADS / 2>(list, have, k, best, most, l->wave_count, &l->taken);
    if (have <= most) return have;
  }
  __syncthreads();
  have = radix_select<T, THREADS>(xr, n, from, k, best, *l);
  __syncthreads();
  return have;
}

// The result of a row from its entries in LDS, at least the k largest of them, and empty slots behind.  Up to 256 entries are
// counted against each other, each by one to eight neighbouring threads; more are sorted (64 rows of which 200 of 131072
// are kept: 32 us, 36 where up to 512 are counted).
template <int THREADS>
__device__ inline void write_result(uint64_t *entries, uint32_t count, size_t row, uint32_t k, float *value, uint32_t *index) {
  if (count <= kCounted) {
    uint32_t sharers = 8u;
    while (sharers > 1u && sharers * count > uint32_t(THREADS)) sharers >>= 1;
    // (each reads four pairs at a time: zeros behind the last entry; the array has room)
    if (threadIdx.x < 64u) entries[count + threadIdx.x] = 0u;
    __syncthreads();
    const uint32_t part = threadIdx.x & (sharers - 1u);
    for (uint32_t i = threadIdx.x / sharers; i < count; i += uint32_t(THREADS) / sharers) {
      const uint64_t own = entries[i];
      uint32_t rank = 0u;
      for (uint32_t j = 2u * part; j < count; j += 8u * sharers) {
        typedef uint64_t pair __attribute__((ext_vector_type(2)));
        pair e[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) e[p] = *reinterpret_cast<const pair *>(&entries[j + 2u * uint32_t(p) * sharers]);
#pragma unroll
        for (int p = 0; p < 4; ++p) rank += (e[p].x > own ? 1u : 0u) + (e[p].y > own ? 1u : 0u);
      }
      for (uint32_t d = 1u; d < sharers; d <<= 1) rank += uint32_t(__shfl_xor(int(rank), int(d), kWave));
      if (part == 0u && rank < k) {
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
  bool near;
};

// What the parts of a row leave for the kernel that joins them.
struct PartResults {
  uint64_t *entries;  // [quota, parts, rows]
  uint32_t *count;    // [parts, rows]
  SoftmaxSum *stats;  // [parts, rows]
  uint32_t quota;
};

// U groups of a thread, `step` apart from g on: what load_tile() does for groups that lie THREADS apart.
template <typename T, int U>
__device__ inline void load_apart(const RowSpan<T> &span, const T *row, uint32_t g, uint32_t step, u32x4 (&q)[U]) {
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t at = min(g + uint32_t(u) * step, span.groups - 1u);
    q[u] = load_stream<0, int(sizeof(T))>(reinterpret_cast<const u32x4 *>(row + size_t(span.first(at))));
  }
}

// A key that at least `share` of a wave's segments reach, from the largest values of each lane's segments, MOST at most, in LDS.
template <typename T, int THREADS, int MOST>
__device__ inline uint32_t key_of_segments(const float *segment, uint32_t segments, uint32_t share) {
  uint32_t key[MOST];
#pragma unroll
  for (int j = 0; j < MOST; ++j) {
    key[j] = uint32_t(j) < segments ? key_of(segment[uint32_t(j) * uint32_t(THREADS) + threadIdx.x]) : 0u;
  }
  uint32_t t = 0u;
#pragma unroll 1
  for (uint32_t bit = 0x80000000u; bit >= LowestBit<T>::value; bit >>= 1) {
    uint32_t reached = 0u;
#pragma unroll
    for (int j = 0; j < MOST; ++j) reached += uint32_t(__popcll(__ballot(key[j] >= (t | bit))));
    if (reached >= share) t |= bit;
  }
  return whole_key<T>(t);
}

// The largest key, but for its low bits, that k of the threads reach, by every wave alike; 0 where fewer hold a key.
template <typename T, int THREADS>
__device__ inline uint32_t key_of_threads(const uint32_t *thread_key, uint32_t k) {
  constexpr int EACH = THREADS / kWave;
  uint32_t key[EACH], t = 0u;
#pragma unroll
  for (int i = 0; i < EACH; ++i) key[i] = thread_key[(threadIdx.x & (kWave - 1)) + uint32_t(i * kWave)];
#pragma unroll
  for (uint32_t bit = 0x80000000u; bit >= LowestBit<T>::value; bit >>= 1) {
    uint32_t reached = 0u;
#pragma unroll
    for (int i = 0; i < EACH; ++i) reached += uint32_t(__popcll(__ballot(key[i] >= (t | bit))));
    if (reached >= k) t |= bit;
  }
  return whole_key<T>(t);
}

// One workgroup a part of a row, which it streams once.  A thread leaves the largest value of each of its segments (up to 16: a
// 16-byte group each, or as many groups as that takes) in LDS.  A threshold that k of the threads' largest values reach (of long
// rows; of short ones every wave finds what its share of k reaches, the least of the waves counts; for large k the
// segments count, not the threads) names the few segments that can hold one of the k largest; these are read again,
// and of their values those that reach the threshold are ranked and written.  (A segment with a NaN has one as its largest
// value and is always read again; its thread counts for nothing in the threshold.)  Rows for which there are too many
// (thousands of ties at the threshold, the largest values all in few segments) are selected from with further passes.
//
// Bound by reading: [2048, 131072] bf16 with the norm 96 us (5.6 TB/s) for k = 1, 99 us (5.4) for k = 64, 231 us for k = 1000,
// whose 1200 candidates are sorted.  A threshold held while the row streams, with a list of what reaches it, took 114 us:
// its branches, barriers and LDS additions cost more than the 75 segments that are read again here.  With 8 segments a
// thread the 64 take 111 us and the 1000 1742, with 32 103 and 294; with two groups of a thread on their way together
// instead of four the 64 take 114.  The threads' threshold instead of the waves' is as quick for random values and eight
// times as quick for rows in falling order.  [512, 131072], k = 64 with the norm, three arrays in turn: f32 62 us of random
// values (44 where one array stays in the last cache), 124 of zeros, 60 in rising order; bf16 33, 79 and 41.
template <typename T, int THREADS, int SHORT, bool NORM>
__global__ __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(THREADS <= 128 && sizeof(T) == 4 ? 5 : 4))) void top_k_kernel(
    uint32_t n, uint32_t rows, size_t stride, uint32_t k, Scale sc, double inv_t, Cut cut, const T *__restrict__ x,
    float *__restrict__ value, uint32_t *__restrict__ index, float *__restrict__ log_norm, PartResults pr) {
  constexpr int W = Group<T>::W;
  constexpr int U = 4;  // groups of a thread together
  constexpr uint32_t WAVES = THREADS / kWave;
  constexpr uint32_t kTile = uint32_t(THREADS) * uint32_t(U);
  constexpr uint32_t kList = uint32_t(kSegments * THREADS) / 2u, kShort = SHORT;  // (twice the largest k it is launched for)
  __shared__ __align__(16) uint64_t list[kList];
  __shared__ __align__(16) uint64_t best[kShort + 64u];
  __shared__ RadixLds radix;
  __shared__ uint32_t wave_key[WAVES];
  __shared__ uint32_t named, listed, taken;
  __shared__ SoftmaxSum sums[WAVES];
  float *const segment = reinterpret_cast<float *>(list);          // [segments, threads]; until the list is filled
  uint32_t *const names = reinterpret_cast<uint32_t *>(best);      // of segments to be read again
  uint32_t *const thread_key = names + kShort;                     // (behind them in the same place)
  const uint32_t wave = threadIdx.x / kWave;
  const uint32_t share = (k + WAVES - 1u) / WAVES;
  const uint64_t items = uint64_t(rows) * cut.parts;
  for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const size_t r = item / cut.parts;
    const uint32_t from = uint32_t(item % cut.parts) * cut.per;
    const uint32_t count = min(cut.per, n - from);
    const T *xr = x + r * stride + from;
    const RowSpan<T> span(count, 0u);
    const uint32_t turns = span.groups / uint32_t(THREADS) + (span.groups % uint32_t(THREADS) != 0u);  // groups of a thread
    const uint32_t tiles = (turns + uint32_t(U) - 1u) / uint32_t(U);
    const bool fine = turns <= uint32_t(kSegments);  // a segment is one group
    const uint32_t span_tiles = (tiles + uint32_t(kSegments) - 1u) / uint32_t(kSegments);
    const uint32_t each = fine ? 1u : span_tiles * uint32_t(U);  // groups of a segment
    const uint32_t segments = (turns + each - 1u) / each;
    const bool near = THREADS > 128 && cut.near && !fine;  // a thread's groups of a tile lie side by side, not THREADS apart
    const uint32_t step = near ? 1u : uint32_t(THREADS), own_first = near ? threadIdx.x * uint32_t(U) : threadIdx.x;
    if (threadIdx.x == 0) named = listed = 0u;
    float top = kMinusInf;
    SoftmaxSum st = {-sc.limit, 0.0f};
    if (span.groups != 0u) {
      u32x4 q[U];
      load_apart<T, U>(span, xr, own_first, step, q);
      float segment_top = kMinusInf;
      uint32_t left = span_tiles;
      float *own = segment + threadIdx.x;
      for (uint32_t base = 0;; base += kTile) {
        float v[U * W];
        u32x4 next[U];
        const bool more = span.groups - base > kTile;
        load_apart<T, U>(span, xr, base + kTile + own_first, step, next);
        unpack_tile<T, U>(q, v);
        if (!more) {
#pragma unroll
          for (int i = 0; i < U * W; ++i) v[i] = base + own_first + uint32_t(i / W) * step < span.groups ? v[i] : kMinusInf;
        }
        float tile_top = kMinusInf;
        if (fine) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            float w[W];
#pragma unroll
            for (int j = 0; j < W; ++j) w[j] = v[u * W + j];
            const float group_top = max_of(kMinusInf, w);
            if (base / uint32_t(THREADS) + uint32_t(u) < uint32_t(kSegments)) own[u * THREADS] = group_top;
            tile_top = larger(tile_top, group_top);
          }
          own += U * THREADS;
        } else {
          tile_top = max_of(kMinusInf, v);
          segment_top = larger(segment_top, tile_top);
          if (--left == 0u || !more) {
            own[0] = segment_top;
            own += THREADS;
            segment_top = kMinusInf;
            left = span_tiles;
          }
        }
        top = larger(top, tile_top);
        if constexpr (NORM) fold_below(st, fmaxf(top, -sc.limit), v, sc.c);
        if (!more) break;
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = next[u];
      }
    }
    // (up to half of the threads: their largest values instead of the segments', 1.4 times k values reach what they give)
    uint32_t low;
    if (THREADS > 128 && k <= uint32_t(THREADS) / 2u) {
      thread_key[threadIdx.x] = key_of(top);
      __syncthreads();
      low = key_of_threads<T, THREADS>(thread_key, k);
    } else {
      const uint32_t t = share <= uint32_t(kWave / 2) ? key_reached_by<T>(key_of(top), share)
                                                      : key_of_segments<T, THREADS, THREADS == 64 ? 2 * U : kSegments>(segment, segments, share);
      if ((threadIdx.x & (kWave - 1)) == 0) wave_key[wave] = t;
      __syncthreads();
      low = wave_key[0];
#pragma unroll
      for (uint32_t w = 1; w < WAVES; ++w) low = min(low, wave_key[w]);
    }
    const float least = low < kLowestKey ? -__FLT_MAX__ : value_of(low);
    uint32_t marked = 0u;
#pragma unroll 4
    for (uint32_t j = 0; j < segments; ++j) marked |= uint32_t(!(segment[j * uint32_t(THREADS) + threadIdx.x] < least)) << j;
    if (k == 0u) marked = 0u;  // (the norm alone)
    uint32_t place = reserve(&named, uint32_t(__popc(marked)));
    for (; marked != 0u && place < kShort; marked &= marked - 1u) {
      names[place++] = (uint32_t(__ffs(int(marked))) - 1u) * uint32_t(THREADS) + threadIdx.x;
    }
    __syncthreads();
    uint32_t have = named <= kShort ? 0u : kNoClass;
    if (have == 0u) {
      const uint32_t again = named * each;
      for (uint32_t base = 0; base < again; base += uint32_t(THREADS)) {
        const uint32_t i = min(base + threadIdx.x, again - 1u);
        const uint32_t name = names[i / each], turn = name / uint32_t(THREADS) * each + i % each;
        const uint32_t thread = name % uint32_t(THREADS), tile = turn / uint32_t(U), u = turn % uint32_t(U);
        const uint32_t g = tile * kTile + (near ? thread * uint32_t(U) + u : thread + u * uint32_t(THREADS));
        const bool mine = base + threadIdx.x < again && g < span.groups;
        float v[W];
        unpack(load_stream<0, int(sizeof(T))>(reinterpret_cast<const u32x4 *>(xr + size_t(span.first(min(g, span.groups - 1u))))), v, x);
        uint32_t reached = 0u;
#pragma unroll
        for (int j = 0; j < W; ++j) reached += mine && v[j] >= least ? 1u : 0u;
        uint32_t place = reserve(&listed, reached);
        if (reached != 0u && place + reached <= kList) {
#pragma unroll
          for (int j = 0; j < W; ++j) {
            if (v[j] >= least) list[place++] = entry_of(key_of(v[j]), from + span.first(g) + uint32_t(j));
          }
        }
      }
      if (span.single(threadIdx.x)) {  // (at most 7: the head is empty)
        const uint32_t at = span.single_at(threadIdx.x);
        const float v = float(xr[at]);
        if (v >= least) {
          const uint32_t place = atomicAdd(&listed, 1u);
          if (place < kList) list[place] = entry_of(key_of(v), from + at);
        }
        if constexpr (NORM) fold_one(st, v, sc.c);
      }
      __syncthreads();
      have = listed;
    } else if (NORM && span.single(threadIdx.x)) {
      fold_one(st, float(xr[span.single_at(threadIdx.x)]), sc.c);
    }
    uint64_t *found = list;
    if (have > kList) {
      have = select_again<T, THREADS>(xr, count, from, top, k, list, kList, best, kShort, &radix);
      found = best;
    } else if (have > kCounted) {
      const uint32_t few = thin_out<T, THREADS, int(kList)>(list, have, k, best, kShort, radix.wave_count, &taken);
      if (few <= kShort) {
        have = few;
        found = best;
      }
    }
    if (cut.parts > 1u && have > pr.quota) {  // more than the part has room for: the k largest of them
      uint32_t size = 2u;
      while (size < have) size <<= 1;
      for (uint32_t i = have + threadIdx.x; i < size; i += THREADS) found[i] = 0u;
      sort_entries<THREADS>(found, size);
      have = k;
    }
    if (cut.parts == 1u) {
      write_result<THREADS>(found, have, r, k, value, index);
      if constexpr (NORM) {
        st = finish_stats<T, THREADS, true>(st, xr, n, sc, sums);
        if (threadIdx.x == 0) log_norm[r] = float(double(st.m) * inv_t + log(double(st.s)));
      }
    } else {
      for (uint32_t i = threadIdx.x; i < have; i += THREADS) pr.entries[item * pr.quota + i] = found[i];
      if (threadIdx.x == 0) pr.count[item] = have;
      if constexpr (NORM) {
        st = finish_stats<T, THREADS, true>(st, xr, count, sc, sums);
        if (threadIdx.x == 0) pr.stats[item] = st;
      }
    }
    __syncthreads();
  }
}

// One workgroup a row: its parts' entries together, thinned, ranked and written.  Latency: 4 to 5 us for some hundred entries.
constexpr uint32_t kJoined = 4096;  // entries of a row's parts at most
template <typename T, bool NORM>
__global__ __launch_bounds__(kBlock) void top_k_join_kernel(uint32_t rows, uint32_t k, Scale sc, double inv_t, uint32_t parts,
                                                            float *__restrict__ value, uint32_t *__restrict__ index,
                                                            float *__restrict__ log_norm, PartResults pr) {
  constexpr uint32_t kShort = 2048;
  __shared__ __align__(16) uint64_t list[kJoined];
  __shared__ __align__(16) uint64_t best[kShort];
  __shared__ uint32_t first[65];
  __shared__ uint32_t wave_count[2 * kBlock / kWave];
  __shared__ uint32_t taken;
  for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
    SoftmaxSum st = {kMinusInf, 0.0f};
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
    const uint32_t few = thin_out<T, kBlock, int(kJoined)>(list, have, k, best, kShort, wave_count, &taken);
    if (few <= kShort) {
      write_result<kBlock>(best, few, r, k, value, index);
    } else {
      write_result<kBlock>(list, have, r, k, value, index);
    }
    if constexpr (NORM) {
      st = join_lanes(st, sc.c);
      if (threadIdx.x == 0) log_norm[r] = float(double(st.m) * inv_t + log(double(st.s)));
    }
    __syncthreads();
  }
}

// Threads of a workgroup: one wave for rows of up to 8 KB (16 where its lanes' largest values give the threshold, k <= 32), 65536
// rows of 1000 bf16, k = 10, 97 us, with two 166; 16384 of 16000 bytes, k = 50, 70 against 64, k = 10 of 8192 32 against 35.
// Two waves for short rows, 8192 of 16000 bf16 64 against 97 us with four; four for long ones, 333 of 50257 halves 18.6
// against 27 with two.  k > 256 takes four and more room in LDS.
constexpr uint32_t kFew = 256;
uint32_t threads_for(uint32_t n, uint32_t k, uint32_t size) {
  if (k <= uint32_t(kWave) && uint64_t(n) * size <= (k <= uint32_t(kWave / 2) ? 16384u : 8192u)) return 64u;
  return n <= 16384u && k <= kFew ? 128u : 256u;
}

// Arrays from this size on, which memory and not the last cache delivers, are read with a thread's four groups side by side: the
// segments read again lie in a quarter of the lines (86 MB of [2048, 131072] bf16, 103 against 99 us; [512, 131072] f32
// 54.8 against 52.0), below it THREADS apart (512 rows of bf16 30.8 against 33.4).
constexpr uint64_t kNearBytes = uint64_t(192) << 20;

// Rows of up to 65536 classes are not cut: the second launch costs more than what it saves (8 rows of 32768 floats 7.1 against 10.0
// us in four parts, 200 of 50257 bf16 11.1 against 16.9, 8 of 65536 bf16 10.8 against 12.2).  Longer ones are, into parts of
// at least 32768 values, no more than bring the launch to eight waves a CU (16 of 131072 bf16 14.0 against 17.2 us in two
// parts and 14.5 in sixteen, 64 of them 14.7 and 16.2 in eight), and with room for three times k entries each among those that
// are joined (a part leaves little more than k).
Cut cut_row(uint32_t n, uint32_t rows, uint32_t k, uint32_t threads, uint32_t size) {
  const bool near = uint64_t(n) * rows * size >= kNearBytes;
  uint64_t parts = uint64_t(device_cu_count()) * (512u / threads) / rows;
  if (parts > n / 32768u) parts = n / 32768u;
  if (parts > 64u) parts = 64u;
  if (k != 0u && parts > kJoined / (3u * k)) parts = kJoined / (3u * k);
  if (parts <= 1u || n <= 65536u) return Cut{1u, n, near};
  const uint64_t per = ((uint64_t(n) + parts - 1u) / parts + 1023u) / 1024u * 1024u;
  return Cut{uint32_t((n + per - 1u) / per), uint32_t(per), near};
}
struct PartBytes {
  size_t entries, stats, counts;
};
PartBytes part_bytes(uint32_t rows, const Cut &cut) {
  const size_t items = size_t(rows) * cut.parts;
  return PartBytes{items * (kJoined / cut.parts) * sizeof(uint64_t), items * sizeof(SoftmaxSum), items * sizeof(uint32_t)};
}

template <typename T, int THREADS, int SHORT, bool NORM>
int launch_top_k(const char *symbol, uint32_t n, uint32_t rows, size_t stride, uint32_t k, float temperature, const T *x,
                 float *value, uint32_t *index, float *log_norm, hipStream_t st) {
  const Cut cut = cut_row(n, rows, k, THREADS, uint32_t(sizeof(T)));
  const uint64_t items = uint64_t(rows) * cut.parts;
  const Scale sc = scale_for(temperature);
  const double inv_t = 1.0 / double(temperature);
  PartResults pr = {nullptr, nullptr, nullptr, kJoined / cut.parts};
  auto *kernel = &top_k_kernel<T, THREADS, SHORT, NORM>;
  if (cut.parts == 1u) {
    return note_launched(symbol, launch(kernel, items, THREADS, 0, st, n, rows, stride, k, sc, inv_t, cut, x, value, index, log_norm, pr));
  }
  const PartBytes bytes = part_bytes(rows, cut);
  const RowsScratch scratch = rows_scratch(st, bytes.entries + bytes.stats + bytes.counts, symbol);
  if (scratch.error != 0) return scratch.error;
  char *at = static_cast<char *>(scratch.lease.ptr);
  pr.entries = reinterpret_cast<uint64_t *>(at);
  pr.stats = reinterpret_cast<SoftmaxSum *>(at + bytes.entries);
  pr.count = reinterpret_cast<uint32_t *>(at + bytes.entries + bytes.stats);
  const hipError_t e = launch(kernel, items, THREADS, 0, st, n, rows, stride, k, sc, inv_t, cut, x, value, index, log_norm, pr);
  if (e != hipSuccess) return note_launched(symbol, e);
  return note_launched(symbol, launch(&top_k_join_kernel<T, NORM>, rows, kBlock, 0, st, rows, k, sc, inv_t, cut.parts,
                                      value, index, log_norm, pr));
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
    auto *launch = &launch_top_k<T, 256, int(kFew) * 2, NORM>;
    if (k > kFew) {
      launch = &launch_top_k<T, 256, int(kMaxSlots) * 2, NORM>;
    } else if (threads_for(dim0, k, uint32_t(sizeof(T))) == 64u) {
      launch = &launch_top_k<T, 64, int(kFew) * 2, NORM>;
    } else if (threads_for(dim0, k, uint32_t(sizeof(T))) == 128u) {
      launch = &launch_top_k<T, 128, int(kFew) * 2, NORM>;
    }
    return launch(symbol, dim0, dim1, pitch, k, temperature, x, value, index, log_norm, st);
  };
  return log_norm != nullptr ? go(std::true_type{}) : go(std::false_type{});
}

}  // namespace

size_t top_k_scratch(uint32_t classes, uint32_t rows, uint32_t k) {
  if (rows == 0u || k > kMaxSlots) return 0u;
  size_t most = 0u;
  for (uint32_t size : {2u, 4u}) {
    const Cut cut = cut_row(classes, rows, k, threads_for(classes, k, size), size);
    const PartBytes b = part_bytes(rows, cut);
    if (cut.parts > 1u && b.entries + b.stats + b.counts > most) most = b.entries + b.stats + b.counts;
  }
  return most;
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
