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

// A row's teacher as the wave knows it that looked at the slots: the log of slot j's probability is
// value * inv_t - shift + log_scale.
struct TeacherRow {
  double shift, log_scale, mass;
  bool any;       // a slot counts
  bool repeated;  // a class is named twice
};

// The slots of a row in LDS.
struct Slots {
  float *p;         // [k]: the probability; 0 for a slot that does not count
  uint32_t *index;  // [k]: its class; kNoClass for a slot that does not count
  float *x;         // [k]: the student's logit, read before dx (which may be x) is written; then the gradient there
  float *old;       // [k]: what dx held (accumulating)
  uint32_t *seen;   // [kSeen], for k > 64: the classes met so far
};
constexpr uint32_t kSeen = 2u * kMaxSlots;
__device__ inline Slots slots_in(uint32_t *lds, uint32_t k) {
  float *f = reinterpret_cast<float *>(lds);
  return Slots{f, lds + k, f + 2u * k, f + 3u * k, lds + 4u * k};
}
uint32_t slot_bytes(uint32_t k) { return 16u * k + (k > uint32_t(kWave) ? 4u * kSeen : 0u); }

// Reads the slots of a row, by one whole wave: x and dx are the row's; only classes in [from, from + count) are kept (the
// mass is the whole row's).
template <typename T, bool ACC>
__device__ inline TeacherRow read_slots(const Teacher &t, size_t row, const T *x, const T *dx, uint32_t n, uint32_t from,
                                        uint32_t count, double inv_t, const Slots &s) {
  const uint32_t lane = threadIdx.x & (kWave - 1);
  const size_t first = row * t.k;
  TeacherRow r = {0.0, 0.0, 0.0, false, false};
  float top = kMinusInf;
  for (uint32_t j = lane; j < t.k; j += kWave) {
    const uint32_t at = t.index[first + j];
    const float v = t.value[first + j];
    const bool counts = at < n && v > kMinusInf;
    s.index[j] = counts ? at : kNoClass;
    s.p[j] = v;
    s.x[j] = counts ? float(x[at]) : 0.0f;
    if (ACC) s.old[j] = counts ? float(dx[at]) : 0.0f;
    if (counts) top = fmaxf(top, v);
  }
  top = wave_max(top);
  r.any = top > kMinusInf;
  if (!r.any) return r;
  r.shift = t.log_norm != nullptr ? double(t.log_norm[row]) : double(top) * inv_t;
  double sum = 0.0;
  for (uint32_t j = lane; j < t.k; j += kWave) {
    const double e = s.index[j] != kNoClass ? exp(double(s.p[j]) * inv_t - r.shift) : 0.0;
    s.p[j] = float(e);
    sum += e;
  }
  sum = wave_sum(sum);
  r.mass = sum;
  if (t.log_norm == nullptr) {
    const float scale = float(1.0 / sum);
    for (uint32_t j = lane; j < t.k; j += kWave) s.p[j] *= scale;
    r.mass = 1.0;
    r.log_scale = -log(sum);
  }
  // whether a class is named twice: among 64 slots by comparing, beyond in a table
  if (t.k <= uint32_t(kWave)) {
    const uint32_t mine = lane < t.k ? s.index[lane] : kNoClass;
    bool twice = false;
    for (uint32_t i = 0; i < t.k; ++i) {
      const uint32_t other = uint32_t(__builtin_amdgcn_readlane(int(mine), int(i)));
      twice |= other == mine && i != lane;
    }
    r.repeated = __any(twice && mine != kNoClass);
  } else {
    for (uint32_t i = lane; i < kSeen; i += kWave) s.seen[i] = kNoClass;
    bool twice = false;
    for (uint32_t j = lane; j < t.k; j += kWave) {
      const uint32_t mine = s.index[j];
      if (mine == kNoClass) continue;
      uint32_t at = (mine * 2654435761u) >> 21;  // (kSeen = 2^11 places, at most half of them taken)
      for (;;) {
        const uint32_t held = atomicCAS(&s.seen[at], kNoClass, mine);
        if (held == kNoClass) break;
        if (held == mine) {
          twice = true;
          break;
        }
        at = (at + 1u) & (kSeen - 1u);
      }
    }
    r.repeated = __any(twice);
  }
  if (from != 0u || count != n) {
    for (uint32_t j = lane; j < t.k; j += kWave) {
      if (s.index[j] - from >= count) s.index[j] = kNoClass;  // (below `from` the difference wraps)
    }
  }
  return r;
}

// The row's loss from its slots in LDS, by the wave that read them.
__device__ inline float slots_loss(const Teacher &t, size_t row, SoftmaxSum st, double inv_t, const TeacherRow &tr, const Slots &s) {
  if (!tr.any) return 0.0f;
  const double log_s = log(double(st.s));
  double loss = 0.0;
  for (uint32_t j = threadIdx.x & (kWave - 1); j < t.k; j += kWave) {
    const float p = s.p[j];
    if (s.index[j] == kNoClass || p == 0.0f) continue;  // (a slot without mass adds nothing, whatever the student says)
    const double lp = double(t.value[row * t.k + j]) * inv_t - tr.shift + tr.log_scale;
    loss += double(p) * (lp - ((double(s.x[j]) - double(st.m)) * inv_t - log_s));
  }
  return float(wave_sum(loss));
}

// The row's loss straight from memory, by one whole wave.
template <typename T>
__device__ inline float row_loss(const Teacher &t, size_t row, const T *x, uint32_t n, SoftmaxSum st, double inv_t) {
  const uint32_t lane = threadIdx.x & (kWave - 1);
  const size_t first = row * t.k;
  float top = kMinusInf;
  for (uint32_t j = lane; j < t.k; j += kWave) {
    if (t.counts(first + j, n)) top = fmaxf(top, t.value[first + j]);
  }
  top = wave_max(top);
  if (!(top > kMinusInf)) return 0.0f;
  // with e_k = exp(a_k): loss = sum e_k (a_k - ln q_k) where the norm is given, else that over sum e_k, less its log
  const double shift = t.log_norm != nullptr ? double(t.log_norm[row]) : double(top) * inv_t;
  const double log_s = log(double(st.s));
  double mass = 0.0, loss = 0.0;
  for (uint32_t j = lane; j < t.k; j += kWave) {
    if (!t.counts(first + j, n)) continue;
    const double a = double(t.value[first + j]) * inv_t - shift, e = exp(a);
    const double lq = (double(float(x[t.index[first + j]])) - double(st.m)) * inv_t - log_s;
    if (e != 0.0) loss += e * (a - lq);  // (a slot without mass adds nothing, whatever the student says)
    mass += e;
  }
  loss = wave_sum(loss);
  if (t.log_norm == nullptr) {
    mass = wave_sum(mass);
    loss = loss / mass - log(mass);
  }
  return float(loss);
}

constexpr int kUnroll = 4;  // 16-byte groups of a thread on their way together

// A part of a row: rows are cut into `parts` of `per` values (whole 16-byte groups) where there are too few to fill the
// GPU.
struct Parts {
  uint32_t parts, per;
  __device__ uint32_t first(uint32_t part) const { return part * per; }
  __device__ uint32_t count(uint32_t part, uint32_t n) const { return min(per, n - part * per); }
};

// One workgroup a row: statistics and loss.
template <typename T, int THREADS, int NT>
__global__ __launch_bounds__(THREADS) void distill_kernel(uint32_t n, uint32_t rows, size_t stride, Scale sc, double inv_t,
                                                          const T *__restrict__ x, Teacher t, float *__restrict__ loss,
                                                          float *__restrict__ row_max, float *__restrict__ row_sum) {
  __shared__ SoftmaxSum lds[THREADS / kWave];
  for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T *xr = x + r * stride;
    const SoftmaxSum st =
        finish_stats<T, THREADS>(stream_stats<T, THREADS, kUnroll, NT>(RowSpan<T>(n, 0u), xr, sc), xr, n, sc, lds);
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

// One workgroup a part of a row: its statistics, to partial[row * parts + part].
template <typename T>
__global__ __launch_bounds__(kBlock) void part_stats_kernel(uint32_t n, uint32_t rows, size_t stride, Scale sc, Parts ps,
                                                            const T *__restrict__ x, SoftmaxSum *__restrict__ partial) {
  __shared__ SoftmaxSum lds[kBlock / kWave];
  const uint64_t items = uint64_t(rows) * ps.parts;
  for (uint64_t i = blockIdx.x; i < items; i += gridDim.x) {
    const uint32_t r = uint32_t(i / ps.parts), part = uint32_t(i % ps.parts);
    const RowSpan<T> span(ps.count(part, n), 0u);
    const SoftmaxSum st = block_merge<kBlock / kWave>(
        stream_stats<T, kBlock, kUnroll, 0>(span, x + size_t(r) * stride + ps.first(part), sc), sc.c, lds);
    if (threadIdx.x == 0) partial[i] = st;
  }
}

// The parts of a row merged, by a whole workgroup whose waves all do the same.
template <typename T, int THREADS>
__device__ inline SoftmaxSum join_parts(const SoftmaxSum *partial, uint32_t parts, const T *row, uint32_t n, Scale sc, float *lds) {
  SoftmaxSum st = {-sc.limit, 0.0f};
  for (uint32_t i = threadIdx.x & (kWave - 1); i < parts; i += kWave) st = merge(st, partial[i], sc.c);
  st = wave_merge(st, sc.c);
  if (measured(st.m, sc)) return SoftmaxSum{st.m, true_sum(st, sc.c)};
  return plain_stats<T, THREADS>(row, n, sc.c, lds);
}

// One wave a row: the parts' statistics joined, and the loss.
template <typename T>
__global__ __launch_bounds__(kWave) void distill_join_kernel(uint32_t n, uint32_t rows, size_t stride, Scale sc, double inv_t,
                                                             uint32_t parts, const T *__restrict__ x, Teacher t,
                                                             const SoftmaxSum *__restrict__ partial, float *__restrict__ loss,
                                                             float *__restrict__ row_max, float *__restrict__ row_sum) {
  __shared__ float lds[1];
  for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const SoftmaxSum st = join_parts<T, kWave>(partial + r * parts, parts, x + r * stride, n, sc, lds);
    const float l = row_loss(t, r, x + r * stride, n, st, inv_t);
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

// The single values of a span.
template <typename T, int THREADS, bool ACC>
__device__ inline void single_grad(const RowSpan<T> &span, const T *x, T *dx, const Dense &d) {
#pragma unroll 1
  for (uint32_t i = threadIdx.x; span.single(i); i += THREADS) {
    const uint32_t at = span.single_at(i);
    float v = any_term(float(x[at]), d);
    if (ACC) v += float(dx[at]);
    dx[at] = T(v);
  }
}

// The dense part of dx over a span, streamed.  Every thread reads and writes its own groups only, in turn, so dx
// may be x.
template <typename T, int THREADS, int U, bool ACC, int NT, bool FAST>
__device__ inline void stream_groups(const RowSpan<T> &span, const T *x, T *dx, const Dense &d) {
  constexpr int W = Group<T>::W;
  constexpr uint32_t kTile = uint32_t(THREADS) * uint32_t(U);
  if (span.groups == 0u) return;
  u32x4 q[U];
  load_tile<T, THREADS, U, 0>(span, x, threadIdx.x, q);
  for (uint32_t base = 0;; base += kTile) {
    const uint32_t g = base + threadIdx.x;
    u32x4 old[U], next[U];
    const bool more = span.groups - base > kTile;
    if (ACC) load_tile<T, THREADS, U, 0>(span, dx, g, old);
    load_tile<T, THREADS, U, 0>(span, x, g + kTile, next);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[W], o[W];
      unpack(q[u], v, x);
      if (ACC) unpack(old[u], o, x);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        v[j] = FAST ? fast_term(v[j], d) : any_term(v[j], d);
        if (ACC) v[j] += o[j];
      }
      const uint32_t at = g + uint32_t(u) * uint32_t(THREADS);
      if (at < span.groups) store_group<NT, int(sizeof(T))>(dx + size_t(span.first(at)), pack(v, dx));
    }
    if (!more) break;
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = next[u];
  }
}
template <typename T, int THREADS, bool ACC, int NT>
__device__ inline void stream_grad(const RowSpan<T> &span, const T *x, T *dx, const Dense &d) {
  single_grad<T, THREADS, ACC>(span, x, dx, d);
  if (d.fast) {
    stream_groups<T, THREADS, kUnroll, ACC, NT, true>(span, x, dx, d);
  } else {
    stream_groups<T, THREADS, kUnroll, ACC, 0, false>(span, x, dx, d);
  }
}

// The gradient at the classes that slots name, into slots.x, by the wave that read the slots.
__device__ inline void slot_grads(uint32_t k, SoftmaxSum st, double inv_t, double w, const TeacherRow &tr, const Slots &s) {
  if (!tr.any) return;
  for (uint32_t j = threadIdx.x & (kWave - 1); j < k; j += kWave) {
    if (s.index[j] == kNoClass) continue;
    const double q = exp((double(s.x[j]) - double(st.m)) * inv_t) / double(st.s);
    double p = double(s.p[j]);
    if (tr.repeated) {  // all of the class's mass, added in slot order whichever of its slots does it
      p = 0.0;
      for (uint32_t i = 0; i < k; ++i) p += s.index[i] == s.index[j] ? double(s.p[i]) : 0.0;
    }
    s.x[j] = float(w * (tr.mass * q - p));
  }
}
// ... and from there to dx.  A class is stored by the wave that stored the 16-byte group it lies in (threads take groups in
// turn, `held` groups first where a kernel keeps that many in registers), so that a wave's own order of stores decides.
// Slots that name one class write the same value.
template <typename T, int THREADS, bool ACC>
__device__ inline void store_slots(uint32_t k, T *dx, uint32_t from, const RowSpan<T> &span, uint32_t held, const Slots &s) {
#pragma unroll 1
  for (uint32_t j = threadIdx.x & (kWave - 1); j < k; j += kWave) {
    if (s.index[j] == kNoClass) continue;
    const uint32_t at = s.index[j] - from, end = span.head + span.groups * uint32_t(RowSpan<T>::W);
    uint32_t turn;
    if (at < span.head || at >= end) {
      turn = at < span.head ? at : at - end + span.head;
    } else {
      turn = (at - span.head) / uint32_t(RowSpan<T>::W);
      if (turn >= held) turn -= held;
    }
    if (turn % uint32_t(THREADS) / kWave == threadIdx.x / kWave) dx[from + at] = T(ACC ? s.old[j] + s.x[j] : s.x[j]);
  }
}

// What the wave that reads the slots leaves for the others.
struct RowShared {
  float mass;
  int any;
};

// One workgroup a part of a row.
template <typename T, int THREADS, bool ACC, int NT>
__global__ __launch_bounds__(THREADS) void distill_bwd_kernel(uint32_t n, uint32_t rows, size_t stride, Scale sc, double inv_t,
                                                              Parts ps, const float *__restrict__ dy, const T *x, Teacher t,
                                                              const float *__restrict__ row_max,
                                                              const float *__restrict__ row_sum, T *dx) {
  extern __shared__ uint32_t slot_lds[];
  __shared__ RowShared rs;
  const Slots slots = slots_in(slot_lds, t.k);
  const uint64_t items = uint64_t(rows) * ps.parts;
  for (uint64_t i = blockIdx.x; i < items; i += gridDim.x) {
    const size_t r = i / ps.parts;
    const uint32_t part = uint32_t(i % ps.parts);
    const uint32_t from = ps.first(part), count = ps.count(part, n);
    const T *xr = x + r * stride;
    T *dxr = dx + r * stride;
    const SoftmaxSum st = {row_max[r], row_sum[r]};
    const double w = double(dy[r]) * inv_t;
    if (threadIdx.x < uint32_t(kWave)) {
      const TeacherRow tr = read_slots<T, ACC>(t, r, xr, dxr, n, from, count, inv_t, slots);
      if (threadIdx.x == 0) rs = RowShared{float(tr.mass), tr.any};
      slot_grads(t.k, st, inv_t, w, tr, slots);
    }
    __syncthreads();
    const Dense d = dense_of(st, sc, float(w), rs.mass, rs.any != 0);
    const RowSpan<T> span(count, values_to_line(dxr + from));
    if (!ACC || d.any) stream_grad<T, THREADS, ACC, NT>(span, xr + from, dxr + from, d);
    if (d.any) store_slots<T, THREADS, ACC>(t.k, dxr, from, span, 0xffffffffu, slots);
    __syncthreads();
  }
}

// Loss and gradient, one workgroup a row: the first G groups of each streaming thread stay in registers from the statistics
// to the gradient, so that x is read once (what lies behind them is streamed a second time).  The
// slots belong to a wave of their own: their 64-bit exponentials and logarithms would spill the held registers of a
// wave that streams, and take about as long as a small row.
template <typename T, int S, int G, int NT>
__global__ __launch_bounds__(S + kWave) __attribute__((amdgpu_waves_per_eu(4))) void distill_held_kernel(
    uint32_t n, uint32_t rows, size_t stride, Scale sc, double inv_t, const T *x, Teacher t, const float *__restrict__ dy,
    float *__restrict__ loss, float *__restrict__ row_max, float *__restrict__ row_sum, T *dx) {
  constexpr int W = Group<T>::W;
  constexpr int THREADS = S + kWave;
  constexpr int WAVES = S / kWave;
  constexpr uint32_t kHeld = uint32_t(S) * uint32_t(G);
  extern __shared__ uint32_t slot_lds[];
  __shared__ SoftmaxSum parts[WAVES];
  __shared__ float plain_lds[WAVES + 1];
  __shared__ RowShared rs;
  const Slots slots = slots_in(slot_lds, t.k);
  // the row's statistics, by every wave alike
  auto joined = [&](const T *xr) {
    const SoftmaxSum st = lane_merge<WAVES>(parts, sc.c);
    if (measured(st.m, sc)) return SoftmaxSum{st.m, true_sum(st, sc.c)};
    return plain_stats<T, THREADS>(xr, n, sc.c, plain_lds);
  };
  if (threadIdx.x >= uint32_t(S)) {
    for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
      const T *xr = x + r * stride;
      const TeacherRow tr = read_slots<T, false>(t, r, xr, dx + r * stride, n, 0u, n, inv_t, slots);
      if (threadIdx.x == uint32_t(S)) rs = RowShared{float(tr.mass), tr.any};
      const double w = double(dy[r]) * inv_t;
      __syncthreads();  // 1: the parts and the mass are there
      const SoftmaxSum st = joined(xr);
      const float l = slots_loss(t, r, st, inv_t, tr, slots);
      if (threadIdx.x == uint32_t(S)) {
        loss[r] = l;
        row_max[r] = st.m;
        row_sum[r] = st.s;
      }
      slot_grads(t.k, st, inv_t, w, tr, slots);
      __syncthreads();  // 2: the slots' gradients are there
      __syncthreads();  // 3: and stored
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
      for (int u = 0; u < G; ++u) q[u] = xb.load<0>(mine, uint32_t(u) * kStep);
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
    single_grad<T, S, false>(span, xr, dxr, d);
    if (d.fast) {
#pragma unroll 1
      for (uint32_t g = kHeld + threadIdx.x; g < span.groups; g += S) {
        float v[W];
        unpack(load_stream<0, int(sizeof(T))>(reinterpret_cast<const u32x4 *>(xr + size_t(span.first(g)))), v, x);
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = fast_term(v[j], d);
        store_group<0, int(sizeof(T))>(dxr + size_t(span.first(g)), pack(v, dx));
      }
      const GroupBuffer db(dxr + span.head, min(span.groups, kHeld));
#pragma unroll
      for (int u = 0; u < G; ++u) {
        float v[W];
        unpack(q[u], v, x);
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = fast_term(v[j], d);
        db.store<NT>(pack(v, dx), mine, uint32_t(u) * kStep);
      }
    } else {
#pragma unroll 1
      for (uint32_t g = threadIdx.x; g < span.groups; g += S) {
        float v[W];
        unpack(load_stream<0, int(sizeof(T))>(reinterpret_cast<const u32x4 *>(xr + size_t(span.first(g)))), v, x);
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = any_term(v[j], d);
        store_group<0, int(sizeof(T))>(dxr + size_t(span.first(g)), pack(v, dx));
      }
    }
    __syncthreads();  // 2
    if (d.any) store_slots<T, S, false>(t.k, dxr, 0u, span, kHeld, slots);
    __syncthreads();  // 3
  }
}

// The same for short rows, one wave a row.
template <typename T, int G, int NT>
__global__ __launch_bounds__(kWave) __attribute__((amdgpu_waves_per_eu(4))) void distill_wave_kernel(
    uint32_t n, uint32_t rows, size_t stride, Scale sc, double inv_t, const T *x, Teacher t, const float *__restrict__ dy,
    float *__restrict__ loss, float *__restrict__ row_max, float *__restrict__ row_sum, T *dx) {
  constexpr int W = Group<T>::W;
  extern __shared__ uint32_t slot_lds[];
  __shared__ SoftmaxSum lds[1];
  const Slots slots = slots_in(slot_lds, t.k);
  for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T *xr = x + r * stride;
    T *dxr = dx + r * stride;
    const RowSpan<T> span(n, values_to_line(dxr));
    u32x4 q[G];
    if (span.groups != 0u) load_tile<T, kWave, G, 0>(span, xr, threadIdx.x, q);
    const TeacherRow tr = read_slots<T, false>(t, r, xr, dxr, n, 0u, n, inv_t, slots);
    const double w = double(dy[r]) * inv_t;
    SoftmaxSum st = {-sc.limit, 0.0f};
    for (uint32_t i = threadIdx.x; span.single(i); i += kWave) fold_one(st, float(xr[span.single_at(i)]), sc.c);
    if (span.groups != 0u) {
      float v[G * W];
      unpack_tile<T, G>(q, v);
      mask_tile<T, kWave, G>(span, threadIdx.x, kMinusInf, v);
      fold(st, v, sc.c);
    }
    st = finish_stats<T, kWave>(st, xr, n, sc, lds);
    const float l = slots_loss(t, r, st, inv_t, tr, slots);
    if (threadIdx.x == 0) {
      loss[r] = l;
      row_max[r] = st.m;
      row_sum[r] = st.s;
    }
    slot_grads(t.k, st, inv_t, w, tr, slots);
    const Dense d = dense_of(st, sc, float(w), float(tr.mass), tr.any);
    single_grad<T, kWave, false>(span, xr, dxr, d);
#pragma unroll
    for (int u = 0; u < G; ++u) {
      const uint32_t at = uint32_t(u) * kWave + threadIdx.x;
      float v[W];
      unpack(q[u], v, x);
#pragma unroll
      for (int j = 0; j < W; ++j) v[j] = any_term(v[j], d);
      if (at < span.groups) store_group<NT, int(sizeof(T))>(dxr + size_t(span.first(at)), pack(v, dx));
    }
    if (d.any) store_slots<T, kWave, false>(t.k, dxr, 0u, span, 0xffffffffu, slots);
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

template <typename T>
int check_arrays(const char *symbol, const Shape &s, const T *x, const Teacher &t, std::initializer_list<const void *> needed) {
  if (s.n != 0u && (x == nullptr || misaligned(x))) return refuse(symbol, "the logits are missing or not aligned to their type");
  if (t.k != 0u && (t.value == nullptr || t.index == nullptr)) return refuse(symbol, "the teacher's slots are missing");
  for (const void *p : needed) {
    if (p == nullptr) return refuse(symbol, "an array is missing");
  }
  return 0;
}

uint32_t grid_for(uint64_t items) { return items < (1u << 24) ? uint32_t(items) : (1u << 24); }

// Parts of at least one tile of a workgroup (kBlock * kUnroll groups), no more than bring the launch to `target`
// workgroups.
template <typename T>
Parts cut_rows(const Shape &s, uint32_t target) {
  const uint32_t tile = uint32_t(kBlock * kUnroll * Group<T>::W);
  uint64_t parts = (uint64_t(target) + s.rows - 1u) / s.rows;
  if (parts > s.n / tile) parts = s.n / tile;
  if (parts <= 1u) return Parts{1u, s.n};
  const uint64_t unit = 1024;  // parts start whole 128-byte lines into a row
  const uint64_t per = ((uint64_t(s.n) + parts - 1u) / parts + unit - 1u) / unit * unit;
  return Parts{uint32_t((s.n + per - 1u) / per), uint32_t(per < s.n ? per : s.n)};
}

template <typename T>
int distill(const char *symbol, uint32_t dim0, uint32_t dim1, uint32_t stride, float temperature, const T *x, const Teacher &t,
            float *loss, float *row_max, float *row_sum, CUstream_st *stream) {
  Shape s;
  if (const int e = prepare(symbol, dim0, dim1, stride, t.k, temperature, s)) return e;
  if (dim1 == 0u) return 0;
  if (const int e = check_arrays(symbol, s, x, t, {loss, row_max, row_sum})) return e;
  const hipStream_t st = as_stream(stream);
  const Parts ps = cut_rows<T>(s, 1024u);
  if (ps.parts > 1u) {
    ScratchLease scratch = acquire_scratch(st, size_t(s.rows) * ps.parts * sizeof(SoftmaxSum), symbol);
    if (!scratch.ptr) return int(hipErrorOutOfMemory);
    SoftmaxSum *partial = static_cast<SoftmaxSum *>(scratch.ptr);
    part_stats_kernel<T><<<grid_for(uint64_t(s.rows) * ps.parts), kBlock, 0, st>>>(s.n, s.rows, s.stride, s.sc, ps, x, partial);
    distill_join_kernel<T><<<grid_for(s.rows), kWave, 0, st>>>(s.n, s.rows, s.stride, s.sc, s.inv_t, ps.parts, x, t, partial, loss,
                                                             row_max, row_sum);
  } else if (size_t(s.n) * sizeof(T) <= 16384u) {
    distill_kernel<T, kWave, 0><<<grid_for(s.rows), kWave, 0, st>>>(s.n, s.rows, s.stride, s.sc, s.inv_t, x, t, loss, row_max,
                                                                  row_sum);
  } else {
    distill_kernel<T, kBlock, 0><<<grid_for(s.rows), kBlock, 0, st>>>(s.n, s.rows, s.stride, s.sc, s.inv_t, x, t, loss, row_max,
                                                                    row_sum);
  }
  note_launch(symbol);
  return 0;
}

template <typename T, bool ACC, int NT>
void launch_bwd(const Shape &s, const float *dy, const T *x, const Teacher &t, const float *row_max, const float *row_sum, T *dx,
                hipStream_t st) {
  const Parts ps = cut_rows<T>(s, 2048u);
  const uint32_t grid = grid_for(uint64_t(s.rows) * ps.parts);
  if (size_t(s.n) * sizeof(T) <= 16384u) {
    distill_bwd_kernel<T, kWave, ACC, NT><<<grid, kWave, slot_bytes(t.k), st>>>(s.n, s.rows, s.stride, s.sc, s.inv_t, ps, dy, x, t,
                                                                               row_max, row_sum, dx);
  } else {
    distill_bwd_kernel<T, kBlock, ACC, NT><<<grid, kBlock, slot_bytes(t.k), st>>>(s.n, s.rows, s.stride, s.sc, s.inv_t, ps, dy, x,
                                                                                 t, row_max, row_sum, dx);
  }
}

template <typename T, bool ACC>
int distill_bwd(const char *symbol, uint32_t dim0, uint32_t dim1, uint32_t stride, float temperature, const float *dy,
                const T *x, const Teacher &t, const float *row_max, const float *row_sum, T *dx, CUstream_st *stream) {
  Shape s;
  if (const int e = prepare(symbol, dim0, dim1, stride, t.k, temperature, s)) return e;
  if (dim1 == 0u || dim0 == 0u) return 0;
  if (const int e = check_arrays(symbol, s, x, t, {dy, row_max, row_sum, dx})) return e;
  if (misaligned(dx)) return refuse(symbol, "the gradient is not aligned to its type");
  if (stream_policy(s.bytes(sizeof(T)), tuning().nontemporal) & kNtStore) {
    launch_bwd<T, ACC, kNtStore>(s, dy, x, t, row_max, row_sum, dx, as_stream(stream));
  } else {
    launch_bwd<T, ACC, 0>(s, dy, x, t, row_max, row_sum, dx, as_stream(stream));
  }
  note_launch(symbol);
  return 0;
}

template <typename T, int NT>
void launch_fused(const Shape &s, const T *x, const Teacher &t, const float *dy, float *loss, float *row_max, float *row_sum,
                  T *dx, hipStream_t st) {
  const size_t row = size_t(s.n) * sizeof(T);
  auto go = [&](auto kernel, uint32_t threads) {
    kernel<<<grid_for(s.rows), threads, slot_bytes(t.k), st>>>(s.n, s.rows, s.stride, s.sc, s.inv_t, x, t, dy, loss, row_max,
                                                              row_sum, dx);
  };
  if (row <= 4096u) {
    go(distill_wave_kernel<T, 4, NT>, kWave);
  } else if (row <= 18432u) {
    go(distill_held_kernel<T, 192, 6, NT>, 256u);
  } else if (row <= 71680u) {
    go(distill_held_kernel<T, 448, 10, NT>, 512u);
  } else if (row <= 136192u) {
    go(distill_held_kernel<T, 448, 20, NT>, 512u);
  } else {
    go(distill_held_kernel<T, 960, 18, NT>, 1024u);
  }
}

template <typename T>
int distill_fused(const char *symbol, uint32_t dim0, uint32_t dim1, uint32_t stride, float temperature, const T *x,
                  const Teacher &t, const float *dy, float *loss, float *row_max, float *row_sum, T *dx, CUstream_st *stream) {
  Shape s;
  if (const int e = prepare(symbol, dim0, dim1, stride, t.k, temperature, s)) return e;
  if (dim1 == 0u) return 0;
  if (const int e = check_arrays(symbol, s, x, t, {dy, loss, row_max, row_sum})) return e;
  if (dim0 != 0u && (dx == nullptr || misaligned(dx))) return refuse(symbol, "the gradient is missing or not aligned to its type");
  if (((reinterpret_cast<uintptr_t>(x) - reinterpret_cast<uintptr_t>(dx)) & 3u) != 0u) {
    // 16-bit arrays that lie an odd number of elements apart: buffer accesses ask for 4-byte alignment of both
    const int e = distill<T>(symbol, dim0, dim1, stride, temperature, x, t, loss, row_max, row_sum, stream);
    return e != 0 ? e : distill_bwd<T, false>(symbol, dim0, dim1, stride, temperature, dy, x, t, row_max, row_sum, dx, stream);
  }
  if (stream_policy(s.bytes(sizeof(T)), tuning().nontemporal) & kNtStore) {
    launch_fused<T, kNtStore>(s, x, t, dy, loss, row_max, row_sum, dx, as_stream(stream));
  } else {
    launch_fused<T, 0>(s, x, t, dy, loss, row_max, row_sum, dx, as_stream(stream));
  }
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
