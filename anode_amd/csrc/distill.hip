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

namespace anode {
namespace {

struct Teacher {
  const float *value;
  const uint32_t *index;
  const float *log_norm;  // null: the slots are the whole distribution
  uint32_t k;
  __device__ bool counts(size_t at, uint32_t n) const { return index[at] < n && value[at] > kMinusInf; }
};

// A row's teacher as the wave knows it that looked at the slots: slot j's probability is exp(value * inv_t - shift) * scale.
struct TeacherRow {
  double shift, scale, mass;
  bool any;  // a slot counts
};

// The slots of a row in LDS.  A streaming thread finds those that lie in its groups by a list of its own, and the turns of its
// that have one by a bit mask, so that it takes their part off the values while it still has them in registers.
struct Slots {
  double *p;        // [k]: the probability
  double *sum;      // [k]: where a class is named twice, the probabilities of a leader and of the slots that follow it
  float *x;         // [k]: the student's logit
  float *off;       // [k]: the teacher's logit; then what is taken off the gradient of its class
  uint32_t *index;  // [k]: the class; kNoClass for a slot that does not count
  uint32_t *next;   // [k]: a slot's leader; then the next slot of the same thread, or kNoClass
  uint32_t *head;   // [threads]: a thread's first slot, or kNoClass
  uint32_t *turns;  // [threads]: bit i for a slot in the thread's groups of turn i, i + 32, ...
  volatile uint16_t *seen;  // [kSeen]: slots' numbers, at the places that their classes give
};
constexpr uint32_t kSeen = 2048;  // (the leading 11 bits of a product)
__device__ inline Slots slots_in(double *lds, uint32_t k, uint32_t threads) {
  float *f = reinterpret_cast<float *>(lds + 2u * k);
  uint32_t *u = reinterpret_cast<uint32_t *>(f + 2u * k), *t = u + 2u * k;
  return Slots{lds, lds + k, f, f + k, u, u + k, t, t + threads, reinterpret_cast<volatile uint16_t *>(t + 2u * threads)};
}
uint32_t slot_bytes(uint32_t k, uint32_t threads) { return 32u * k + 8u * threads + 2u * kSeen; }

// Reads the slots of a row, by one whole wave: x is the row, n its length.  LOSS: the student's logits too, which the loss asks for
// and the gradient does not.
template <bool LOSS, typename T>
__device__ inline TeacherRow read_slots(const Teacher &t, size_t row, const T *x, uint32_t n, double inv_t, const Slots &s) {
  const uint32_t lane = threadIdx.x & (kWave - 1);
  const size_t first = row * t.k;
  TeacherRow r = {0.0, 1.0, 0.0, false};
  float top = kMinusInf;
  for (uint32_t j = lane; j < t.k; j += kWave) {
    const uint32_t at = t.index[first + j];
    const float v = t.value[first + j];
    const bool counts = at < n && v > kMinusInf;
    s.index[j] = counts ? at : kNoClass;
    s.off[j] = v;
    if (LOSS) s.x[j] = counts ? float(x[at]) : 0.0f;
    if (counts) top = fmaxf(top, v);
  }
  top = lanes_max(top);
  r.any = top > kMinusInf;
  if (!r.any) return r;
  r.shift = t.log_norm != nullptr ? double(t.log_norm[row]) : double(top) * inv_t;
  double sum = 0.0;
  for (uint32_t j = lane; j < t.k; j += kWave) {
    const double e = s.index[j] != kNoClass ? exp(double(s.off[j]) * inv_t - r.shift) : 0.0;
    s.p[j] = e;
    sum += e;
  }
  sum = lanes_sum(sum);
  r.mass = sum;
  if (t.log_norm == nullptr) {
    r.scale = 1.0 / sum;
    for (uint32_t j = lane; j < t.k; j += kWave) s.p[j] *= r.scale;
    r.mass = 1.0;
  }
  return r;
}

// Finds the leader of every slot that counts, one slot of those that name its class, by the wave that read them, and tells whether
// there is one with followers.  A slot leaves its number at a place of a table that its class gives, and looks whose number
// is there: its leader's, if that names its class.  If not, once more at another place (the slots whose number stands
// are done each time, so this ends).  What the table held before does not matter.
__device__ inline bool find_leaders(uint32_t k, const Slots &s) {
  const uint32_t lane = threadIdx.x & (kWave - 1);
  bool repeated = false;
  uint32_t open = 0u;  // bit i: slot lane + 64 i has no leader yet
  for (uint32_t j = lane, bit = 1u; j < k; j += kWave, bit <<= 1) open |= s.index[j] != kNoClass ? bit : 0u;
  for (uint32_t factor = 2654435761u; __any(open != 0u); factor = (factor * 0x9e3779b1u + 0x7f4a7c16u) | 1u) {
    for (uint32_t j = lane, bit = 1u; j < k; j += kWave, bit <<= 1) {
      if ((open & bit) != 0u) s.seen[(s.index[j] * factor) >> 21] = uint16_t(j);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (uint32_t j = lane, bit = 1u; j < k; j += kWave, bit <<= 1) {
      if ((open & bit) == 0u) continue;
      const uint32_t mine = s.index[j], there = s.seen[(mine * factor) >> 21];
      if (s.index[there] == mine) {
        open &= ~bit;
        s.next[j] = there;
        repeated |= there != j;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  return __any(repeated);
}

// The probabilities of a class that is named more than once, at its leader; added one follower after the other, in slot order.
__device__ inline void add_followers(uint32_t k, const Slots &s) {
  const uint32_t lane = threadIdx.x & (kWave - 1);
  for (uint32_t j = lane; j < k; j += kWave) s.sum[j] = s.p[j];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  for (uint32_t base = 0; base < k; base += kWave) {
    const uint32_t j = base + lane;
    const bool counts = j < k && s.index[min(j, k - 1u)] != kNoClass;
    const uint32_t leader = counts ? s.next[j] : j;
    for (uint64_t rest = __ballot(leader != j); rest != 0u; rest &= rest - 1u) {
      const int at = __ffsll((unsigned long long)rest) - 1;
      const uint32_t to = from_lane(leader, at);
      if (lane == 0u) s.sum[to] += s.p[base + uint32_t(at)];
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// Deals the slots that lie in [from, from + n of the span) of the row to the streaming threads, w times their
// probability each; by the wave that read them.  A class that is named more than once gets all of its mass from one slot.
template <typename T, int THREADS>
__device__ inline void deal_slots(uint32_t k, bool any, const RowSpan<T> &span, uint32_t from, double w, const Slots &s) {
  const uint32_t lane = threadIdx.x & (kWave - 1);
  const uint32_t end = span.head + span.groups * uint32_t(RowSpan<T>::W);
  for (uint32_t i = lane; i < uint32_t(THREADS); i += kWave) {
    s.head[i] = kNoClass;
    s.turns[i] = 0u;
  }
  if (!any) return;
  const bool repeated = find_leaders(k, s);
  if (repeated) add_followers(k, s);
  for (uint32_t j = lane; j < k; j += kWave) {
    const uint32_t at = s.index[j] - from;
    const bool mine = s.index[j] != kNoClass && at < end + span.tail && s.next[j] == j;  // (a class below `from` wraps)
    s.next[j] = kNoClass;
    s.off[j] = float(w * (repeated ? s.sum[j] : s.p[j]));
    if (!mine) continue;
    const bool single = at < span.head || at >= end;
    const uint32_t place = single ? (at < span.head ? at : at - end + span.head) : (at - span.head) / uint32_t(RowSpan<T>::W);
    const uint32_t thread = place % uint32_t(THREADS);
    s.next[j] = atomicExch(&s.head[thread], j);
    if (!single) atomicOr(&s.turns[thread], 1u << (place / uint32_t(THREADS) & 31u));
  }
}

// Takes the slots of the thread's list that lie in the W classes from `first` on off their values.
template <int W>
__device__ inline void take_slots(const Slots &s, uint32_t first, float (&v)[W]) {
  for (uint32_t j = s.head[threadIdx.x]; j != kNoClass; j = s.next[j]) {
    const uint32_t at = s.index[j] - first;
    const float off = s.off[j];
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] -= at == uint32_t(i) ? off : 0.0f;
  }
}

// The row's loss from its slots in LDS, by the wave that read them.
__device__ inline float slots_loss(const Teacher &t, size_t row, SoftmaxSum st, double inv_t, const TeacherRow &tr, const Slots &s) {
  if (!tr.any) return 0.0f;
  const double logs = log(double(st.s) * tr.scale);  // ln S and the logarithm of the probabilities' scale
  double loss = 0.0;
  for (uint32_t j = threadIdx.x & (kWave - 1); j < t.k; j += kWave) {
    const double p = s.p[j];
    if (s.index[j] == kNoClass || p == 0.0) continue;  // (a slot without mass adds nothing, whatever the student says)
    const double lp = double(t.value[row * t.k + j]) * inv_t - tr.shift;
    loss += p * (lp - (double(s.x[j]) - double(st.m)) * inv_t + logs);
  }
  return float(lanes_sum(loss));
}

// A lane's slot of a row: the first 64 slots are asked for before the row is streamed, so that their chain of loads (class,
// logit) is over when the statistics are there.
struct LaneSlot {
  float value, x;
  bool counts;
};
template <typename T>
__device__ inline LaneSlot lane_slot(const Teacher &t, size_t row, const T *x, uint32_t n, uint32_t j) {
  LaneSlot s = {kMinusInf, 0.0f, false};
  if (j < t.k) {
    const uint32_t at = t.index[row * t.k + j];
    s.value = t.value[row * t.k + j];
    s.counts = at < n && s.value > kMinusInf;
    if (s.counts) s.x = float(x[at]);
  }
  return s;
}

// The row's loss straight from memory, by one whole wave; `mine` is its lanes' first slots.
template <typename T>
__device__ inline float row_loss(const Teacher &t, size_t row, const T *x, uint32_t n, SoftmaxSum st, double inv_t, LaneSlot mine) {
  const uint32_t lane = threadIdx.x & (kWave - 1);
  float top = mine.counts ? mine.value : kMinusInf;
  for (uint32_t j = lane + kWave; j < t.k; j += kWave) {
    if (t.counts(row * t.k + j, n)) top = fmaxf(top, t.value[row * t.k + j]);
  }
  top = lanes_max(top);
  if (!(top > kMinusInf)) return 0.0f;
  // with e_k = exp(a_k), M = sum e_k: loss = sum e_k (a_k - (x_k - m) / T) + M ln S where the norm is given, else the sum over M,
  // and ln (S / M)
  const double shift = t.log_norm != nullptr ? double(t.log_norm[row]) : double(top) * inv_t;
  double mass = 0.0, loss = 0.0;
  for (uint32_t j = lane; j < t.k; j += kWave) {
    const LaneSlot s = j == lane ? mine : lane_slot(t, row, x, n, j);
    if (!s.counts) continue;
    const double a = double(s.value) * inv_t - shift, e = exp(a);
    if (e != 0.0) loss += e * (a - (double(s.x) - double(st.m)) * inv_t);  // (a slot without mass adds nothing, whatever the student says)
    mass += e;
  }
  loss = lanes_sum(loss);
  mass = lanes_sum(mass);
  if (mass == 0.0) return 0.0f;
  const double share = t.log_norm != nullptr ? 1.0 : 1.0 / mass, logs = log(double(st.s) * share);
  return float((loss + mass * logs) * share);
}

constexpr int kUnroll = 4;  // 16-byte groups of a thread on their way together

// A part of a row: rows are cut into `parts` of `per` values (whole 16-byte groups) where there are too few to fill the
// GPU.
struct Parts {
  uint32_t parts, per;
  __device__ uint32_t first(uint32_t part) const { return part * per; }
  __device__ uint32_t count(uint32_t part, uint32_t n) const { return min(per, n - part * per); }
};

// One workgroup a row: statistics and loss.  Long rows are bound by reading: 4096 of 131072 bf16 6.0 TB/s, 1001 of 50257 halves 21.6
// us (4.7 TB/s; 3 of them are the launch's beginning and end).  Short ones by the VALU, half of it the slots' 64-bit
// terms: 65536 of 1000 bf16 57 us.
template <typename T, int THREADS, int U>
__global__ __launch_bounds__(THREADS) void distill_kernel(uint32_t n, uint32_t rows, size_t stride, Scale sc, double inv_t,
                                                          const T *__restrict__ x, Teacher t, float *__restrict__ loss,
                                                          float *__restrict__ row_max, float *__restrict__ row_sum) {
  __shared__ SoftmaxSum lds[THREADS / kWave];
  for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T *xr = x + r * stride;
    LaneSlot slot = {};
    if (threadIdx.x < uint32_t(kWave)) slot = lane_slot(t, r, xr, n, threadIdx.x);
    const SoftmaxSum st =
        finish_stats<T, THREADS, false>(stream_stats<T, THREADS, U>(RowSpan<T>(n, 0u), xr, sc), xr, n, sc, lds);
    if (threadIdx.x < uint32_t(kWave)) {
      const float l = row_loss(t, r, xr, n, st, inv_t, slot);
      if (threadIdx.x == 0) {
        loss[r] = l;
        row_max[r] = st.m;
        row_sum[r] = st.s;
      }
    }
  }
}

// One workgroup a part of a row: its statistics, finished, to partial[row * parts + part].  24 rows of 131072 bf16 are 384 parts, 3.9 us, and
// 3.7 for the kernel that joins them: latency.
template <typename T>
__global__ __launch_bounds__(kBlock) void part_stats_kernel(uint32_t n, uint32_t rows, size_t stride, Scale sc, Parts ps,
                                                            const T *__restrict__ x, SoftmaxSum *__restrict__ partial) {
  __shared__ SoftmaxSum lds[kBlock / kWave];
  const uint64_t items = uint64_t(rows) * ps.parts;
  for (uint64_t i = blockIdx.x; i < items; i += gridDim.x) {
    const uint32_t r = uint32_t(i / ps.parts), part = uint32_t(i % ps.parts);
    const T *xp = x + size_t(r) * stride + ps.first(part);
    const uint32_t count = ps.count(part, n);
    const SoftmaxSum st =
        finish_stats<T, kBlock, false>(stream_stats<T, kBlock, kUnroll>(RowSpan<T>(count, 0u), xp, sc), xp, count, sc, lds);
    if (threadIdx.x == 0) partial[i] = st;
  }
}

// The parts of a row joined, by every wave alike: a lane takes every 64th of them, the lanes then meet.
__device__ inline SoftmaxSum join_parts(const SoftmaxSum *partial, uint32_t parts, Scale sc) {
  SoftmaxSum st = {kMinusInf, 0.0f};
  for (uint32_t i = threadIdx.x & (kWave - 1); i < parts; i += kWave) {
    const SoftmaxSum p = partial[i];
    const float m = fmaxf(st.m, p.m), about = m == kMinusInf ? 0.0f : m;
    st.s = st.s * __builtin_amdgcn_exp2f((st.m - about) * sc.c) + p.s * __builtin_amdgcn_exp2f((p.m - about) * sc.c);
    st.m = m;
  }
  return join_lanes(st, sc.c);
}

// One wave a row: the parts' statistics joined, and the loss.
template <typename T>
__global__ __launch_bounds__(kWave) void distill_join_kernel(uint32_t n, uint32_t rows, size_t stride, Scale sc, double inv_t,
                                                             uint32_t parts, const T *__restrict__ x, Teacher t,
                                                             const SoftmaxSum *__restrict__ partial, float *__restrict__ loss,
                                                             float *__restrict__ row_max, float *__restrict__ row_sum) {
  for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const LaneSlot slot = lane_slot(t, r, x + r * stride, n, threadIdx.x);
    const SoftmaxSum st = join_parts(partial + r * parts, parts, sc);
    const float l = row_loss(t, r, x + r * stride, n, st, inv_t, slot);
    if (threadIdx.x == 0) {
      loss[r] = l;
      row_max[r] = st.m;
      row_sum[r] = st.s;
    }
  }
}

// What the dense part of a row's gradient is made of: dx_j = exp2(x_j c - shift) * scale in the fast form.
struct Dense {
  float m, c, shift, scale;
  bool fast;  // else exp2((x - m) * c) * scale, or zeros
  bool any;
};
__device__ inline Dense dense_of(SoftmaxSum st, Scale sc, float w, float mass, bool any) {
  Dense d;
  d.m = st.m;
  d.c = sc.c;
  d.shift = st.m * sc.c;
  d.fast = measured(st.m, sc) && any;
  d.any = any;
  d.scale = w * mass / st.s;
  if (d.fast) d.scale *= __builtin_amdgcn_exp2f(fmaf(-st.m, sc.c, d.shift));
  return d;
}
__device__ inline float fast_term(float x, const Dense &d) { return __builtin_amdgcn_exp2f(fmaf(x, d.c, -d.shift)) * d.scale; }
__device__ inline float any_term(float x, const Dense &d) {
  if (d.fast) return fast_term(x, d);
  return d.any ? __builtin_amdgcn_exp2f((x - d.m) * d.c) * d.scale : 0.0f;
}

// The single values of a span; `at` of the slots' classes counts from the row's start, the span starts at `from`.
template <typename T, int THREADS, bool ACC>
__device__ inline void single_grad(const RowSpan<T> &span, const T *x, T *dx, uint32_t from, const Dense &d, const Slots &slots) {
#pragma unroll 1
  for (uint32_t i = threadIdx.x; span.single(i); i += THREADS) {
    const uint32_t at = span.single_at(i);
    float v[1] = {any_term(float(x[at]), d)};
    if (ACC) v[0] += float(dx[at]);
    take_slots(slots, from + at, v);
    dx[at] = T(v[0]);
  }
}

// The groups of a span, streamed; q holds the thread's first tile already.  Every thread reads and writes its own groups only,
// in turn, so dx may be x.
template <typename T, int THREADS, int U, bool ACC, int NT, bool FAST>
__device__ inline void stream_groups(const RowSpan<T> &span, const T *x, T *dx, uint32_t from, const Dense &d, const Slots &slots,
                                     u32x4 (&q)[U]) {
  constexpr int W = Group<T>::W;
  constexpr uint32_t kTile = uint32_t(THREADS) * uint32_t(U);
  if (span.groups == 0u) return;
  const uint32_t turns = slots.turns[threadIdx.x];
  uint32_t turn = 0u;
  for (uint32_t base = 0;; base += kTile) {
    const uint32_t g = base + threadIdx.x;
    u32x4 old[U], next[U];
    const bool more = span.groups - base > kTile;
    if (ACC) load_tile<T, THREADS, U>(span, dx, g, old);
    load_tile<T, THREADS, U>(span, x, g + kTile, next);
#pragma unroll
    for (int u = 0; u < U; ++u, ++turn) {
      float v[W], o[W];
      unpack(q[u], v, x);
      if (ACC) unpack(old[u], o, x);
      const uint32_t at = g + uint32_t(u) * uint32_t(THREADS);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        v[j] = FAST ? fast_term(v[j], d) : any_term(v[j], d);
        if (ACC) v[j] += o[j];
      }
      if ((turns >> (turn & 31u) & 1u) != 0u) take_slots(slots, from + span.first(at), v);
      if (at < span.groups) store_group<NT, int(sizeof(T))>(dx + size_t(span.first(at)), pack(v, dx));
    }
    if (!more) break;
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = next[u];
  }
}

// What the wave that reads the slots leaves for the others.
struct RowShared {
  float mass;
  int any;
};

// What a pass over the parts of rows left (part_stats_kernel), and where the rows' results go.
struct Joined {
  const SoftmaxSum *partial;  // null: row_max and row_sum are inputs
  float *loss, *row_max, *row_sum;
};

// One workgroup a part of a row.  JOIN: the row's statistics are put together from its parts by every workgroup for itself, and
// the first part's writes them and the loss.  Bound by memory: 1001 rows of 50257 halves 36.0 us (5.6 TB/s read and
// written), 512 of 131072 floats 95 us.
template <typename T, int THREADS, int U, bool ACC, bool JOIN, int NT>
__global__ __launch_bounds__(THREADS) void distill_bwd_kernel(uint32_t n, uint32_t rows, size_t stride, Scale sc, double inv_t,
                                                              Parts ps, const float *__restrict__ dy, const T *x, Teacher t,
                                                              Joined jn, T *dx) {
  extern __shared__ double slot_lds[];
  __shared__ RowShared rs;
  const Slots slots = slots_in(slot_lds, t.k, THREADS);
  const uint64_t items = uint64_t(rows) * ps.parts;
  for (uint64_t i = blockIdx.x; i < items; i += gridDim.x) {
    const size_t r = i / ps.parts;
    const uint32_t part = uint32_t(i % ps.parts);
    const uint32_t from = ps.first(part), count = ps.count(part, n);
    const T *xr = x + r * stride;
    T *dxr = dx + r * stride;
    const RowSpan<T> span(count, values_to_line(dxr + from));
    u32x4 q[U];
    if (span.groups != 0u) load_tile<T, THREADS, U>(span, xr + from, threadIdx.x, q);
    SoftmaxSum st;
    if (JOIN) {
      st = join_parts(jn.partial + r * ps.parts, ps.parts, sc);
    } else {
      st = SoftmaxSum{jn.row_max[r], jn.row_sum[r]};
    }
    const double w = double(dy[r]) * inv_t;
    if (threadIdx.x < uint32_t(kWave)) {
      const TeacherRow tr = read_slots<JOIN>(t, r, xr, n, inv_t, slots);
      if (threadIdx.x == 0) rs = RowShared{float(tr.mass), tr.any};
      deal_slots<T, THREADS>(t.k, tr.any, span, from, w, slots);
      if (JOIN && part == 0u) {
        const float l = slots_loss(t, r, st, inv_t, tr, slots);
        if (threadIdx.x == 0) {
          jn.loss[r] = l;
          jn.row_max[r] = st.m;
          jn.row_sum[r] = st.s;
        }
      }
    }
    __syncthreads();
    const Dense d = dense_of(st, sc, float(w), rs.mass, rs.any != 0);
    if (!ACC || d.any) {
      single_grad<T, THREADS, ACC>(span, xr + from, dxr + from, from, d, slots);
      if (d.fast) {
        stream_groups<T, THREADS, U, ACC, NT, true>(span, xr + from, dxr + from, from, d, slots, q);
      } else {
        stream_groups<T, THREADS, U, ACC, 0, false>(span, xr + from, dxr + from, from, d, slots, q);
      }
    }
    __syncthreads();
  }
}

// Loss and gradient, one workgroup a row: the first G groups of each streaming thread stay in registers from the statistics
// to the gradient, so that x is read once (what lies behind them is streamed a second time).  The slots belong to a wave of
// their own: their 64-bit exponentials and logarithms would spill the held registers of a wave that streams, and take
// about as long as a small row.  [4096, 131072] bf16 407 us, [2048, 32768] f32 100 us, 5.3 TB/s read and written: what bounds it is
// that a CU loads its rows, then stores them.  The same accesses without any arithmetic take 387 us of the first, a flat copy 328;
// two workgroups a CU that hold half of their rows and read the rest twice 475.
template <typename T, int S, int G, int NT>
__global__ __launch_bounds__(S + kWave) __attribute__((amdgpu_waves_per_eu(4))) void distill_held_kernel(
    uint32_t n, uint32_t rows, size_t stride, Scale sc, double inv_t, const T *x, Teacher t, const float *__restrict__ dy,
    float *__restrict__ loss, float *__restrict__ row_max, float *__restrict__ row_sum, T *dx) {
  constexpr int W = Group<T>::W;
  constexpr int THREADS = S + kWave;
  constexpr int WAVES = S / kWave;
  constexpr uint32_t kHeld = uint32_t(S) * uint32_t(G);
  static_assert(G % 2 == 0 && G <= 32, "two groups are folded together; a bit of Slots::turns for each");
  extern __shared__ double slot_lds[];
  __shared__ SoftmaxSum parts[WAVES];
  __shared__ float plain_lds[WAVES + 1];
  __shared__ RowShared rs;
  const Slots slots = slots_in(slot_lds, t.k, S);
  // the row's statistics, by every wave alike
  auto joined = [&](const T *xr) {
    const SoftmaxSum st = lane_merge<WAVES>(parts, sc.c);
    if (measured(st, sc)) return SoftmaxSum{st.m, true_sum(st, sc.c)};
    return plain_stats<T, THREADS, 1>(xr, n, sc.c, plain_lds);
  };
  if (threadIdx.x >= uint32_t(S)) {
    for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
      const T *xr = x + r * stride;
      const TeacherRow tr = read_slots<true>(t, r, xr, n, inv_t, slots);
      if (threadIdx.x == uint32_t(S)) rs = RowShared{float(tr.mass), tr.any};
      deal_slots<T, S>(t.k, tr.any, RowSpan<T>(n, values_to_line(dx + r * stride)), 0u, double(dy[r]) * inv_t, slots);
      __syncthreads();  // 1: the parts, the mass and the lists are there
      const SoftmaxSum st = joined(xr);
      const float l = slots_loss(t, r, st, inv_t, tr, slots);
      if (threadIdx.x == uint32_t(S)) {
        loss[r] = l;
        row_max[r] = st.m;
        row_sum[r] = st.s;
      }
      __syncthreads();  // 2: all of it is done with
    }
    return;
  }
  const uint32_t mine = threadIdx.x * 16u;  // (bytes) the thread's place among a step's groups
  constexpr uint32_t kStep = uint32_t(S) * 16u;
  for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T *xr = x + r * stride;
    T *dxr = dx + r * stride;
    const RowSpan<T> span(n, values_to_line(dxr));
    u32x4 q[G];
    {
      const GroupBuffer xb(xr + span.head, min(span.groups, kHeld));
#pragma unroll
      for (int u = 0; u < G; ++u) q[u] = xb.load(mine, uint32_t(u) * kStep);
    }
    const float w = float(double(dy[r]) * inv_t);
    SoftmaxSum st = {-sc.limit, 0.0f};
#pragma unroll 1
    for (uint32_t g = kHeld + threadIdx.x; g < span.groups; g += S) {
      float v[W];
      unpack(load_stream<0, int(sizeof(T))>(reinterpret_cast<const u32x4 *>(xr + size_t(span.first(g)))), v, x);
      fold(st, v, sc.c);
    }
#pragma unroll 1
    for (uint32_t i = threadIdx.x; span.single(i); i += S) fold_one(st, float(xr[span.single_at(i)]), sc.c);
#pragma unroll
    for (int b = 0; b < G; b += 2) {
      if (span.groups > uint32_t(b) * uint32_t(S)) {
        const u32x4 part[2] = {q[b], q[b + 1]};
        float v[2 * W];
        unpack_tile<T, 2>(part, v);
        if (span.groups < uint32_t(b + 2) * uint32_t(S)) {
          mask_tile<T, S, 2>(span, uint32_t(b) * uint32_t(S) + threadIdx.x, kMinusInf, v);
        }
        fold(st, v, sc.c);
      }
    }
    st = wave_merge(st, sc.c);
    if ((threadIdx.x & (kWave - 1)) == 0) parts[threadIdx.x / kWave] = st;
    __syncthreads();  // 1
    st = joined(xr);
#pragma unroll
    for (int u = 0; u < G; ++u) forget(q[u]);
    const Dense d = dense_of(st, sc, w, rs.mass, rs.any != 0);
    const uint32_t turns = slots.turns[threadIdx.x];
    single_grad<T, S, false>(span, xr, dxr, 0u, d, slots);
    // the groups behind the held ones, or, of a row that the fast form does not measure, all of them
    uint32_t turn = d.fast ? uint32_t(G) : 0u;
#pragma unroll 1
    for (uint32_t g = turn * uint32_t(S) + threadIdx.x; g < span.groups; g += S, ++turn) {
      float v[W];
      unpack(load_stream<0, int(sizeof(T))>(reinterpret_cast<const u32x4 *>(xr + size_t(span.first(g)))), v, x);
#pragma unroll
      for (int j = 0; j < W; ++j) v[j] = any_term(v[j], d);
      if ((turns >> (turn & 31u) & 1u) != 0u) take_slots(slots, span.first(g), v);
      store_group<0, int(sizeof(T))>(dxr + size_t(span.first(g)), pack(v, dx));
    }
    if (d.fast) {
      const GroupBuffer db(dxr + span.head, min(span.groups, kHeld));
#pragma unroll
      for (int u = 0; u < G; ++u) {
        float v[W];
        unpack(q[u], v, x);
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = fast_term(v[j], d);
        if ((turns >> u & 1u) != 0u) take_slots(slots, span.first(uint32_t(u) * uint32_t(S) + threadIdx.x), v);
        db.store<NT>(pack(v, dx), mine, uint32_t(u) * kStep);
      }
    }
    __syncthreads();  // 2
  }
}

// The same for short rows, one wave a row.  Bound by the VALU: 65536 rows of 1000 bf16 116 us, where a copy takes 40; most of a
// wave's 900 instructions are the slots'.
template <typename T, int G, int NT>
__global__ __launch_bounds__(kWave) __attribute__((amdgpu_waves_per_eu(4))) void distill_wave_kernel(
    uint32_t n, uint32_t rows, size_t stride, Scale sc, double inv_t, const T *x, Teacher t, const float *__restrict__ dy,
    float *__restrict__ loss, float *__restrict__ row_max, float *__restrict__ row_sum, T *dx) {
  constexpr int W = Group<T>::W;
  extern __shared__ double slot_lds[];
  __shared__ SoftmaxSum lds[1];
  const Slots slots = slots_in(slot_lds, t.k, kWave);
  for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T *xr = x + r * stride;
    T *dxr = dx + r * stride;
    const RowSpan<T> span(n, values_to_line(dxr));
    u32x4 q[G];
    if (span.groups != 0u) load_tile<T, kWave, G>(span, xr, threadIdx.x, q);
    const double w = double(dy[r]) * inv_t;
    const TeacherRow tr = read_slots<true>(t, r, xr, n, inv_t, slots);
    deal_slots<T, kWave>(t.k, tr.any, span, 0u, w, slots);
    SoftmaxSum st = {-sc.limit, 0.0f};
    for (uint32_t i = threadIdx.x; span.single(i); i += kWave) fold_one(st, float(xr[span.single_at(i)]), sc.c);
    if (span.groups != 0u) {
      float v[G * W];
      unpack_tile<T, G>(q, v);
      mask_tile<T, kWave, G>(span, threadIdx.x, kMinusInf, v);
      fold(st, v, sc.c);
    }
    st = finish_stats<T, kWave, false>(st, xr, n, sc, lds);
    const float l = slots_loss(t, r, st, inv_t, tr, slots);
    if (threadIdx.x == 0) {
      loss[r] = l;
      row_max[r] = st.m;
      row_sum[r] = st.s;
    }
    __syncthreads();
    const Dense d = dense_of(st, sc, float(w), float(tr.mass), tr.any);
    const uint32_t turns = slots.turns[threadIdx.x];
    single_grad<T, kWave, false>(span, xr, dxr, 0u, d, slots);
#pragma unroll
    for (int u = 0; u < G; ++u) {
      const uint32_t at = uint32_t(u) * kWave + threadIdx.x;
      float v[W];
      unpack(q[u], v, x);
#pragma unroll
      for (int j = 0; j < W; ++j) v[j] = any_term(v[j], d);
      if ((turns >> u & 1u) != 0u) take_slots(slots, span.first(at), v);
      if (at < span.groups) store_group<NT, int(sizeof(T))>(dxr + size_t(span.first(at)), pack(v, dx));
    }
    __syncthreads();
  }
}

// ---- host side ----

struct Shape {
  uint32_t n, rows;
  size_t stride;
  Scale sc;
  double inv_t;
  size_t bytes(size_t element) const { return size_t(n) * rows * element; }
};

int prepare(const char *symbol, uint32_t dim0, uint32_t dim1, uint32_t stride, uint32_t k, float temperature, Shape &s) {
  if (const int e = check_rows(symbol, dim0, stride, k, temperature)) return e;
  s = Shape{dim0, dim1, size_t(stride != 0u ? stride : dim0), scale_for(temperature), 1.0 / double(temperature)};
  return 0;
}

// Whether the rows of two arrays lie in each other without being the same ones.  (Rows of one padded array may lie between the
// rows of another.)
template <typename T>
bool tangled(const T *x, const T *dx, const Shape &s) {
  if (x == dx || s.n == 0u) return false;
  const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(dx);
  const size_t apart = a < b ? b - a : a - b, row = size_t(s.n) * sizeof(T), step = s.stride * sizeof(T);
  const size_t rows = apart / step, into = apart % step;
  return (rows < s.rows && into < row) || (rows + 1u < s.rows && step - into < row);
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

// Bytes of a row up to which one wave streams it alone: 8192 rows of 16 KB 30.7 us for the loss and 82 with the gradient, with four
// waves 40 and 101; of 4096 rows of 32 KB the loss takes 29.7 and 30.1 us, with the gradient 84 and 77.  Where the rows
// do not fill the GPU the gradient takes four waves from 4 KB on: 1024 rows of 16 KB 15.6 against 22 us, 2048 rows
// 27.5 against 25.8.
constexpr size_t kWaveRow = 16384;
// Up to here it has two groups of a thread on their way together, and room for more waves on the SIMD: 65536 rows of 1000 bf16 61.6
// against 77 us for the loss and 133 against 170 with the gradient, of 1000 floats 73 and 80, 165 and 189; rows of 8000
// bytes 17.4 against 16.7.  (The fused call holds two groups a thread up to half of it: 118 against 144 us.)
constexpr size_t kShortRow = 4096;

// Bytes of a row that the workgroups of the fused call hold in registers: those of a wave, and of five of distill_held_kernel; a
// sixth, the widest, takes the rest.  At each border the smaller one is the quicker, with rows of bf16: 77 against 182 us
// (32768 rows of 4 KB), 82 against 86 (16384 of 12 KB), 57 against 143 (8192 of 18 KB), 62 against 74 (4096 of 40 KB),
// 58 against 66 (2048 of 70 KB), 59 against 68 (1024 of 140 KB).
constexpr size_t kHeldByWave = size_t(kWave) * 4u * 16u;
constexpr size_t kHeldBy64 = 64u * 12u * 16u, kHeldBy192 = 192u * 6u * 16u;
constexpr size_t kHeldBy448[3] = {448u * 6u * 16u, 448u * 10u * 16u, 448u * 20u * 16u};

// Few rows that only the widest workgroup would hold go in parts, each read a second time for the gradient: 14.8 against 18.7
// us for 24 rows of 131072 bf16 logits.  At 64 rows the two are even, and shorter rows are quicker on one CU each (16
// rows of 32768: 13.7 against 11.2 us).
constexpr uint32_t kFewRows = 32;

// Parts of at least one tile of a workgroup (kBlock * kUnroll groups), no more than bring the launch to kWanted workgroups:
// four a CU (1001 rows of 50257 halves: loss and gradient 58.6 us whole, 66.3 us in two and three parts).
constexpr uint32_t kWanted = 1024;
Parts cut_rows(uint32_t n, uint32_t rows, uint32_t width) {
  const uint32_t tile = uint32_t(kBlock * kUnroll) * width;
  uint64_t parts = kWanted / rows;
  if (parts > n / tile) parts = n / tile;
  if (parts <= 1u) return Parts{1u, n};
  const uint64_t unit = 1024;  // parts start whole 128-byte lines into a row
  const uint64_t per = ((uint64_t(n) + parts - 1u) / parts + unit - 1u) / unit * unit;
  return Parts{uint32_t((n + per - 1u) / per), uint32_t(per < n ? per : n)};
}
template <typename T>
Parts cut_rows(const Shape &s) {
  return cut_rows(s.n, s.rows, uint32_t(Group<T>::W));
}
size_t partial_bytes(uint32_t rows, const Parts &ps) { return size_t(rows) * ps.parts * sizeof(SoftmaxSum); }

// Classes of a row up to which the loss alone takes it whole: the launch that joins the parts costs more (200 rows of 50257 bf16 7.9
// against 11.4 us, 24 of 65536 7.1 against 9.3, of floats 8.0 and 9.3; 24 of 131072 10.4 against 9.3, of floats 15.5 and 9.1).
constexpr uint32_t kWholeLoss = 65536;

template <typename T>
int distill(const char *symbol, uint32_t dim0, uint32_t dim1, uint32_t stride, float temperature, const T *x, const Teacher &t,
            float *loss, float *row_max, float *row_sum, CUstream_st *stream) {
  Shape s;
  if (const int e = prepare(symbol, dim0, dim1, stride, t.k, temperature, s)) return e;
  if (dim1 == 0u) return 0;
  if (const int e = check_arrays(symbol, s, x, t, {loss, row_max, row_sum})) return e;
  const hipStream_t st = as_stream(stream);
  const Parts ps = cut_rows<T>(s);
  if (ps.parts > 1u && s.n > kWholeLoss) {
    const RowsScratch scratch = rows_scratch(st, partial_bytes(s.rows, ps), symbol);
    if (scratch.error != 0) return scratch.error;
    SoftmaxSum *partial = static_cast<SoftmaxSum *>(scratch.lease.ptr);
    const hipError_t e =
        launch(&part_stats_kernel<T>, uint64_t(s.rows) * ps.parts, kBlock, 0, st, s.n, s.rows, s.stride, s.sc, ps, x, partial);
    if (e != hipSuccess) return note_launched(symbol, e);
    return note_launched(symbol, launch(&distill_join_kernel<T>, s.rows, kWave, 0, st, s.n, s.rows, s.stride, s.sc, s.inv_t,
                                        ps.parts, x, t, partial, loss, row_max, row_sum));
  }
  auto go = [&](auto *kernel, uint32_t threads) {
    return note_launched(symbol, launch(kernel, s.rows, threads, 0, st, s.n, s.rows, s.stride, s.sc, s.inv_t, x, t, loss, row_max,
                                        row_sum));
  };
  const size_t row = size_t(s.n) * sizeof(T);
  if (row <= kShortRow) return go(&distill_kernel<T, kWave, 2>, kWave);
  if (row <= kWaveRow) return go(&distill_kernel<T, kWave, kUnroll>, kWave);
  return go(&distill_kernel<T, kBlock, kUnroll>, kBlock);
}

template <typename T, bool ACC, int NT>
hipError_t launch_bwd(const Shape &s, const float *dy, const T *x, const Teacher &t, const float *row_max, const float *row_sum, T *dx,
                hipStream_t st) {
  const Parts ps = cut_rows<T>(s);
  const uint64_t items = uint64_t(s.rows) * ps.parts;
  const Joined jn = {nullptr, nullptr, const_cast<float *>(row_max), const_cast<float *>(row_sum)};  // (read only)
  auto go = [&](auto *kernel, uint32_t threads) {
    return launch(kernel, items, threads, slot_bytes(t.k, threads), st, s.n, s.rows, s.stride, s.sc, s.inv_t, ps, dy, x, t, jn, dx);
  };
  const size_t row = size_t(s.n) * sizeof(T);
  if (row <= kShortRow) return go(&distill_bwd_kernel<T, kWave, 2, ACC, false, NT>, kWave);
  if (row <= kWaveRow && s.rows > kWanted) return go(&distill_bwd_kernel<T, kWave, kUnroll, ACC, false, NT>, kWave);
  return go(&distill_bwd_kernel<T, kBlock, kUnroll, ACC, false, NT>, kBlock);
}

template <typename T, bool ACC>
int distill_bwd(const char *symbol, uint32_t dim0, uint32_t dim1, uint32_t stride, float temperature, const float *dy,
                const T *x, const Teacher &t, const float *row_max, const float *row_sum, T *dx, CUstream_st *stream) {
  Shape s;
  if (const int e = prepare(symbol, dim0, dim1, stride, t.k, temperature, s)) return e;
  if (dim1 == 0u || dim0 == 0u) return 0;
  if (const int e = check_arrays(symbol, s, x, t, {dy, row_max, row_sum, dx})) return e;
  if (misaligned(dx)) return refuse(symbol, "the gradient is not aligned to its type");
  if (tangled<T>(x, dx, s)) return refuse(symbol, "the gradient's rows lie across the logits'");
  const bool nt = (stream_policy(s.bytes(sizeof(T)), tuning().nontemporal) & kNtStore) != 0;
  auto *go = nt ? &launch_bwd<T, ACC, kNtStore> : &launch_bwd<T, ACC, 0>;
  return note_launched(symbol, go(s, dy, x, t, row_max, row_sum, dx, as_stream(stream)));
}

template <typename T, int NT>
hipError_t launch_fused(const Shape &s, const T *x, const Teacher &t, const float *dy, float *loss, float *row_max, float *row_sum,
                  T *dx, hipStream_t st) {
  const size_t row = size_t(s.n) * sizeof(T);
  auto go = [&](auto *kernel, uint32_t threads) {
    const uint32_t streaming = threads > uint32_t(kWave) ? threads - uint32_t(kWave) : threads;
    return launch(kernel, s.rows, threads, slot_bytes(t.k, streaming), st, s.n, s.rows, s.stride, s.sc, s.inv_t, x, t, dy, loss,
                  row_max, row_sum, dx);
  };
  if (row <= kHeldByWave / 2u) return go(&distill_wave_kernel<T, 2, NT>, kWave);
  if (row <= kHeldByWave) return go(&distill_wave_kernel<T, 4, NT>, kWave);
  if (row <= kHeldBy64) return go(&distill_held_kernel<T, 64, 12, NT>, 128u);
  if (row <= kHeldBy192) return go(&distill_held_kernel<T, 192, 6, NT>, 256u);
  if (row <= kHeldBy448[0]) return go(&distill_held_kernel<T, 448, 6, NT>, 512u);
  if (row <= kHeldBy448[1]) return go(&distill_held_kernel<T, 448, 10, NT>, 512u);
  if (row <= kHeldBy448[2]) return go(&distill_held_kernel<T, 448, 20, NT>, 512u);
  return go(&distill_held_kernel<T, 960, 18, NT>, 1024u);
}

template <typename T>
int distill_fused(const char *symbol, uint32_t dim0, uint32_t dim1, uint32_t stride, float temperature, const T *x,
                  const Teacher &t, const float *dy, float *loss, float *row_max, float *row_sum, T *dx, CUstream_st *stream) {
  Shape s;
  if (const int e = prepare(symbol, dim0, dim1, stride, t.k, temperature, s)) return e;
  if (dim1 == 0u) return 0;
  if (const int e = check_arrays(symbol, s, x, t, {dy, loss, row_max, row_sum})) return e;
  if (dim0 != 0u && (dx == nullptr || misaligned(dx))) return refuse(symbol, "the gradient is missing or not aligned to its type");
  if (tangled<T>(x, dx, s)) return refuse(symbol, "the gradient's rows lie across the logits'");
  if (((reinterpret_cast<uintptr_t>(x) - reinterpret_cast<uintptr_t>(dx)) & 3u) != 0u) {
    // 16-bit arrays that lie an odd number of elements apart: buffer accesses ask for 4-byte alignment of both
    const int e = distill<T>(symbol, dim0, dim1, stride, temperature, x, t, loss, row_max, row_sum, stream);
    return e != 0 ? e : distill_bwd<T, false>(symbol, dim0, dim1, stride, temperature, dy, x, t, row_max, row_sum, dx, stream);
  }
  const Parts ps = cut_rows<T>(s);
  // (not where dx is x: a part would overwrite logits that the other parts' workgroups still gather)
  if (s.rows <= kFewRows && size_t(s.n) * sizeof(T) > kHeldBy448[2] && ps.parts > 1u && x != dx) {
    const hipStream_t st = as_stream(stream);
    const RowsScratch scratch = rows_scratch(st, partial_bytes(s.rows, ps), symbol);
    if (scratch.error != 0) return scratch.error;
    SoftmaxSum *partial = static_cast<SoftmaxSum *>(scratch.lease.ptr);
    const uint64_t items = uint64_t(s.rows) * ps.parts;
    const hipError_t e = launch(&part_stats_kernel<T>, items, kBlock, 0, st, s.n, s.rows, s.stride, s.sc, ps, x, partial);
    if (e != hipSuccess) return note_launched(symbol, e);
    return note_launched(symbol, launch(&distill_bwd_kernel<T, kBlock, kUnroll, false, true, 0>, items, kBlock, slot_bytes(t.k, kBlock), st,
                                        s.n, s.rows, s.stride, s.sc, s.inv_t, ps, dy, x, t, Joined{partial, loss, row_max, row_sum}, dx));
  }
  const bool nt = (stream_policy(s.bytes(sizeof(T)), tuning().nontemporal) & kNtStore) != 0;
  auto *go = nt ? &launch_fused<T, kNtStore> : &launch_fused<T, 0>;
  return note_launched(symbol, go(s, x, t, dy, loss, row_max, row_sum, dx, as_stream(stream)));
}

}  // namespace

size_t distill_scratch(uint32_t classes, uint32_t rows) {
  if (classes == 0u || rows == 0u) return 0u;
  size_t most = 0u;
  for (uint32_t width : {4u, 8u}) {
    const Parts ps = cut_rows(classes, rows, width);
    if (ps.parts > 1u && partial_bytes(rows, ps) > most) most = partial_bytes(rows, ps);
  }
  return most;
}
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
