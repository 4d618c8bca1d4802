// Verification of drafted tokens against the target's probabilities, from given random numbers.  No kernel of the
// reference corresponds to it; it takes the probabilities as the row softmax entry points write them.
//
// Of a sequence, drafted token i with target probability p_i and draft probability q_i is taken while u_i q_i < p_i
// (with probability min(1, p / q) for a uniform u).  After the first one that is not taken the token is drawn from the
// target's row less the draft's, max(0, p - q); after all of them from the target's next row.  Drawn is the smallest
// class whose running sum of weights exceeds u times their total.  Whole numbers come out, so the products and the
// sums are in 64 bits: a running sum of 131072 weights in 32 bits is off by more than many a weight.
#include "class_rows.hpp"

namespace anode {
namespace {

constexpr int kDrawThreads = 1024;
constexpr int kDrawWaves = kDrawThreads / kWave;

struct Drafts {
  uint32_t n, drafted;       // classes; drafted tokens of a sequence at most
  const float *target;       // [n, drafted + 1, sequences]
  const float *draft;        // [n, drafted, sequences], or null: every draft is a point mass
  const uint32_t *token;     // [drafted, sequences]
  const uint32_t *length;    // [sequences], or null: all of them hold `drafted`
  const float *accept;       // [drafted, sequences]
};

// The weights a token is drawn from: those of a target row, less a draft's row or one class.  What is not greater
// than zero (a NaN among it) weighs nothing.
struct Weights {
  const float *p, *q;
  uint32_t without;
  __device__ double of(uint32_t j, float pj, float qj) const {
    double w = double(pj);
    if (q != nullptr) w -= double(qj);
    return w > 0.0 && j != without ? w : 0.0;
  }
};

// The four weights of a 16-byte group of the row, in class order.
__device__ inline void group_weights(const RowGroups<float> &rg, const Weights &ws, uint32_t g, double (&w)[4]) {
  float p[4], q[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  load_group<float, 0>(rg, ws.p, g, 0.0f, p);
  if (ws.q != nullptr) load_group<float, 0>(rg, ws.q, g, 0.0f, q);
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = ws.of(rg.first(g) + uint32_t(j), p[j], q[j]);
}

// Drafted tokens that sequence b takes, and how many it holds; by one whole wave.
__device__ inline uint32_t taken_tokens(const Drafts &d, size_t b, uint32_t &length) {
  const uint32_t lane = threadIdx.x & (kWave - 1);
  length = d.length != nullptr ? min(d.length[b], d.drafted) : d.drafted;
  for (uint32_t base = 0; base < length; base += kWave) {
    const uint32_t i = base + lane;
    bool refused = false;
    if (i < length) {
      const size_t at = b * d.drafted + i;
      const uint32_t token = d.token[at];
      refused = true;
      if (token < d.n) {
        const double p = double(d.target[(b * (size_t(d.drafted) + 1u) + i) * d.n + token]);
        const double q = d.draft != nullptr ? double(d.draft[at * d.n + token]) : 1.0;
        refused = !(double(d.accept[at]) * q < p);  // (exact: the product of two 24-bit numbers)
      }
    }
    const uint64_t out = __ballot(refused);
    if (out != 0u) return base + uint32_t(__ffsll((unsigned long long)out)) - 1u;
  }
  return length;
}

// One workgroup a sequence.  Every wave sums a contiguous part of the row; the part in which the running sum passes
// the border is summed again, every thread a contiguous piece, and the piece in which it passes is walked.
__global__ __launch_bounds__(kDrawThreads) void verify_draft_kernel(Drafts d, uint32_t sequences, const float *__restrict__ pick,
                                                                    uint32_t *__restrict__ out, uint32_t *__restrict__ accepted) {
  __shared__ double part[kDrawWaves];
  __shared__ uint32_t s_taken, s_length, s_drawn, s_first;
  const uint32_t lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const RowGroups<float> rg(d.n, 0u);
  for (size_t b = blockIdx.x; b < sequences; b += gridDim.x) {
    if (wave == 0) {
      uint32_t length;
      const uint32_t taken = taken_tokens(d, b, length);
      if (lane == 0) {
        s_taken = taken;
        s_length = length;
        s_drawn = kNoClass;
      }
    }
    __syncthreads();
    const uint32_t taken = s_taken;
    const bool refused = taken < s_length;
    Weights ws;
    ws.p = d.target + (b * (size_t(d.drafted) + 1u) + taken) * d.n;
    ws.q = refused && d.draft != nullptr ? d.draft + (b * d.drafted + taken) * size_t(d.n) : nullptr;
    ws.without = refused && d.draft == nullptr ? d.token[b * d.drafted + taken] : kNoClass;
    const uint32_t each = (rg.groups + kDrawWaves - 1u) / kDrawWaves;  // groups of a wave
    double total = 0.0;
    for (int turn = 0; turn < 2; ++turn) {
      double sum = 0.0;
      const uint32_t end = min(rg.groups, (wave + 1u) * each);
      for (uint32_t g = wave * each + lane; g < end; g += kWave) {
        double w[4];
        group_weights(rg, ws, g, w);
        sum += (w[0] + w[1]) + (w[2] + w[3]);
      }
      sum = wave_sum(sum);
      if (lane == 0) part[wave] = sum;
      __syncthreads();
      total = 0.0;
      for (int w = 0; w < kDrawWaves; ++w) total += part[w];
      if (total > 0.0 || !refused) break;
      // nothing is left of the difference (the target equals the draft there): the target's row itself
      ws.q = nullptr;
      ws.without = kNoClass;
      __syncthreads();
    }
    const double border = double(pick[b]) * total;
    // the part in which the running sum passes the border; where none does (u of 1 and more, a NaN) the last that weighs
    uint32_t in = kNoClass, last = kNoClass;
    double before = 0.0, before_last = 0.0;
    for (uint32_t w = 0; w < uint32_t(kDrawWaves); ++w) {
      if (!(part[w] > 0.0)) continue;
      last = w;
      before_last = before;
      if (before + part[w] > border) {
        in = w;
        break;
      }
      before += part[w];
    }
    if (in == kNoClass) {
      in = last;
      before = before_last;
    }
    __syncthreads();
    if (in != kNoClass) {
      const uint32_t lo = min(rg.groups, in * each), hi = min(rg.groups, lo + each);
      const uint32_t piece = (hi - lo + kDrawThreads - 1u) / kDrawThreads;
      const uint32_t g0 = min(hi, lo + threadIdx.x * piece), g1 = min(hi, g0 + piece);
      double own = 0.0;
      for (uint32_t g = g0; g < g1; ++g) {
        double w[4];
        group_weights(rg, ws, g, w);
        own += (w[0] + w[1]) + (w[2] + w[3]);
      }
      double upto = own;
#pragma unroll
      for (int off = 1; off < kWave; off <<= 1) {
        const double o = __shfl_up(upto, off, kWave);
        if (int(lane) >= off) upto += o;
      }
      if (lane == kWave - 1) part[wave] = upto;
      if (threadIdx.x == 0) s_first = kNoClass;
      __syncthreads();
      for (uint32_t w = 0; w < wave; ++w) before += part[w];
      // the first piece that passes the border, or else the last that weighs
      const bool weighs = own > 0.0;
      const bool passes = weighs && before + upto > border;
      if (passes) atomicMin(&s_first, threadIdx.x);
      __syncthreads();
      if (s_first == kNoClass) {
        __syncthreads();
        if (threadIdx.x == 0) s_first = 0u;
        __syncthreads();
        if (weighs) atomicMax(&s_first, threadIdx.x);
        __syncthreads();
      }
      if (threadIdx.x == s_first) {
        double run = before + (upto - own);
        uint32_t drawn = kNoClass;
        bool done = false;
        for (uint32_t g = g0; g < g1 && !done; ++g) {
          double w[4];
          group_weights(rg, ws, g, w);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (!done && w[j] > 0.0) {
              drawn = rg.first(g) + uint32_t(j);
              run += w[j];
              done = run > border;
            }
          }
        }
        s_drawn = drawn;
      }
      __syncthreads();
    }
    if (threadIdx.x == 0) accepted[b] = taken;
    for (uint32_t i = threadIdx.x; i <= d.drafted; i += kDrawThreads) {
      out[b * (size_t(d.drafted) + 1u) + i] = i < taken ? d.token[b * d.drafted + i] : i == taken ? s_drawn : kNoClass;
    }
    __syncthreads();
  }
}

}  // namespace
}  // namespace anode

ANODE_EXPORT int anode_gpu_verify_draft_packed_f32(uint32_t dim0, uint32_t dim1, uint32_t dim2, const float *target,
                                                   const float *draft, const uint32_t *draft_token, const uint32_t *draft_length,
                                                   const float *accept, const float *pick, uint32_t *token, uint32_t *accepted,
                                                   const KernelConfig *, CUstream_st *stream) {
  using namespace anode;
  if (dim2 == 0u) return 0;
  if (dim0 != 0u && target == nullptr) return refuse(__func__, "the target's probabilities are missing");
  if (dim1 != 0u && (draft_token == nullptr || accept == nullptr)) return refuse(__func__, "the drafted tokens are missing");
  if (pick == nullptr || token == nullptr || accepted == nullptr) return refuse(__func__, "an array is missing");
  if (dim1 == 0xffffffffu) return refuse(__func__, "more drafted tokens than an index holds");
  const uint32_t grid = dim2 < (1u << 24) ? dim2 : (1u << 24);
  const Drafts d = {dim0, dim1, target, draft, draft_token, draft_length, accept};
  verify_draft_kernel<<<grid, kDrawThreads, 0, as_stream(stream)>>>(d, dim2, pick, token, accepted);
  note_launch(__func__);
  return 0;
}
