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

constexpr int kDrawThreads = 256;
constexpr uint32_t kDrawWaves = kDrawThreads / kWave;
constexpr uint32_t kBlockGroups = 512;  // 16-byte groups (2048 classes) of a row that are summed together: eight a lane
// Rows of up to 32 blocks (65536 classes) are drawn from in one launch, a workgroup a sequence; longer rows are spread over the
// GPU first and drawn from by a second kernel.  At 32768 classes 9.4 against 11.7 us for 200 sequences and 8.1 against
// 10.0 for 16, at 50257 14.6 against 17.0 and 11.2 against 11.3 for 64, at 65536 13.2 against 15.6 and 12.2 against 11.8;
// at 131072 18.5 against 10.2 us for 16 and 153 against 136 us for 1024.
constexpr uint32_t kMostHeld = 32;

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
  __device__ static double weight(double w) { return fmax(w, 0.0); }
  __device__ double of(uint32_t j, float pj, float qj) const {
    double w = double(pj);
    if (q != nullptr) w -= double(qj);
    return j != without ? weight(w) : 0.0;
  }
};

// The rows that sequence b's token is drawn from once `taken` of its drafted tokens are taken.
__device__ inline Weights weights_of(const Drafts &d, size_t b, uint32_t taken, bool refused) {
  Weights ws;
  ws.p = d.target + (b * (size_t(d.drafted) + 1u) + taken) * d.n;
  ws.q = refused && d.draft != nullptr ? d.draft + (b * d.drafted + taken) * size_t(d.n) : nullptr;
  ws.without = refused && d.draft == nullptr ? d.token[b * d.drafted + taken] : kNoClass;
  return ws;
}

// Sums of one block of a row: what is left of the target after the draft, and the target itself, from which the token is
// drawn where nothing is left.
struct BlockSum {
  double rest, whole;
};

// One block by a whole wave, groups lane, lane + 64, ... of it.
template <bool DRAFT, int NT>
__device__ inline BlockSum sum_block(const RowGroups<float> &rg, const Weights &ws, uint32_t lo) {
  constexpr int U = 4;
  const uint32_t lane = threadIdx.x & (kWave - 1);
  BlockSum s = {0.0, 0.0};
  const uint32_t end = min(rg.groups - lo, kBlockGroups);            // groups of the block
  const uint32_t whole_end = min(rg.n / 4u - lo, kBlockGroups);      // (the row's last group can be shorter)
  if (whole_end != 0u) {
#pragma unroll
    for (uint32_t half = 0; half < kBlockGroups; half += uint32_t(U) * kWave) {
      u32x4 p[U], q[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t at = lo + min(half + uint32_t(u) * kWave + lane, whole_end - 1u);
        p[u] = load_stream<NT>(reinterpret_cast<const u32x4 *>(ws.p + size_t(at) * 4u));
        if (DRAFT) q[u] = load_stream<NT>(reinterpret_cast<const u32x4 *>(ws.q + size_t(at) * 4u));
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t at = half + uint32_t(u) * kWave + lane;
        double rest[4], whole[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float pj = __uint_as_float(p[u][j]);
          whole[j] = Weights::weight(double(pj));
          rest[j] = DRAFT ? Weights::weight(double(pj) - double(__uint_as_float(q[u][j])))
                          : ((lo + at) * 4u + uint32_t(j) != ws.without ? whole[j] : 0.0);
        }
        if (at < whole_end) {
          s.rest += (rest[0] + rest[1]) + (rest[2] + rest[3]);
          s.whole += (whole[0] + whole[1]) + (whole[2] + whole[3]);
        }
      }
    }
  }
  if (whole_end < end && lane < rg.n % 4u) {
    const uint32_t j = (lo + whole_end) * 4u + lane;
    s.rest += ws.of(j, ws.p[j], DRAFT ? ws.q[j] : 0.0f);
    s.whole += Weights::weight(double(ws.p[j]));
  }
  s.rest = lanes_sum(s.rest);
  s.whole = lanes_sum(s.whole);
  return s;
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

// The first lane whose running sum passes the border, of those that weigh; or else (u of 1 and more, a NaN, the last
// step's rounding) the last that weighs; -1 where none does.
__device__ inline int lane_at(double own, double upto, double border) {
  const uint64_t weighs = __ballot(own > 0.0);
  const uint64_t passes = __ballot(own > 0.0 && upto > border);
  if (passes != 0u) return __ffsll((unsigned long long)passes) - 1;
  return weighs != 0u ? 63 - __clzll((long long)weighs) : -1;
}

// The drawn class, by one whole wave from the sums of the row's blocks: the block in which the running sum passes the border,
// the lane's eight groups of it in which it does, and the class; nothing leaves the registers.
__device__ __forceinline__ uint32_t draw_token(const RowGroups<float> &rg, Weights ws, uint32_t blocks, const BlockSum *sums, double u) {
  constexpr int kOwn = int(kBlockGroups) / kWave;
  const uint32_t lane = threadIdx.x & (kWave - 1);
  const uint32_t each = (blocks + kWave - 1u) / kWave;  // blocks of a lane
  const uint32_t b0 = min(blocks, lane * each), b1 = min(blocks, b0 + each);
  BlockSum mine = {0.0, 0.0};
  for (uint32_t i = b0; i < b1; ++i) {
    const BlockSum s = sums[i];
    mine.rest += s.rest;
    mine.whole += s.whole;
  }
  double own = mine.rest;
  double upto = lanes_upto(own), total = from_lane(upto, kWave - 1);
  const bool left = total > 0.0;
  if (!left) {
    // nothing is left of the difference (the target equals the draft there): the target's row itself
    ws.q = nullptr;
    ws.without = kNoClass;
    own = mine.whole;
    upto = lanes_upto(own);
    total = from_lane(upto, kWave - 1);
  }
  const double border = u * total;
  const int at = lane_at(own, upto, border);
  if (at < 0) return kNoClass;
  uint32_t block = from_lane(b0, at);
  double before = from_lane(upto - own, at);
  if (each > 1u) {  // among that lane's blocks in turn
    const uint32_t end = from_lane(b1, at);
    double run = before;
    for (uint32_t i = block; i < end; ++i) {
      const BlockSum s = sums[i];
      const double w = left ? s.rest : s.whole;
      if (w > 0.0) {
        block = i;
        before = run;
        if (run + w > border) break;
      }
      run += w;
    }
  }
  // among the lanes' eight groups of the block each, which lie side by side
  const uint32_t g0 = block * kBlockGroups + lane * uint32_t(kOwn);
  const uint32_t whole = rg.n / 4u;
  const float *qs = ws.q != nullptr ? ws.q : ws.p;
  own = 0.0;
  if (whole != 0u) {
#pragma unroll
    for (int half = 0; half < kOwn; half += 4) {
      // (a group past the row's whole ones reads the last of them again: no branch, so the loads are on their way together)
      u32x4 p[4], q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const size_t at = size_t(min(g0 + uint32_t(half + i), whole - 1u)) * 4u;
        p[i] = load_stream<0>(reinterpret_cast<const u32x4 *>(ws.p + at));
        q[i] = load_stream<0>(reinterpret_cast<const u32x4 *>(qs + at));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t g = g0 + uint32_t(half + i);
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < 4; ++j) sum += ws.of(g * 4u + uint32_t(j), __uint_as_float(p[i][j]), __uint_as_float(q[i][j]));
        own += g < whole ? sum : 0.0;
      }
    }
  }
  if (whole >= g0 && whole - g0 < uint32_t(kOwn)) {  // the row's last, shorter group is this lane's
    for (uint32_t j = whole * 4u; j < rg.n; ++j) own += ws.of(j, ws.p[j], qs[j]);
  }
  upto = before + lanes_upto(own);
  const int run = lane_at(own, upto, border);
  if (run < 0) return kNoClass;  // (not reached: the block weighs)
  // among those 32 classes, one a lane
  before = from_lane(upto - own, run);
  const uint32_t first = (block * kBlockGroups + uint32_t(run) * uint32_t(kOwn)) * 4u, j = first + lane;
  own = lane < 4u * uint32_t(kOwn) && j < rg.n ? ws.of(j, ws.p[j], qs[j]) : 0.0;
  upto = before + lanes_upto(own);
  const int last = lane_at(own, upto, border);
  return last < 0 ? kNoClass : first + uint32_t(last);
}

// What a sequence gets, by one whole wave.
__device__ inline void write_tokens(const Drafts &d, size_t b, uint32_t taken, uint32_t drawn, uint32_t *out, uint32_t *accepted) {
  const uint32_t lane = threadIdx.x & (kWave - 1);
  if (lane == 0u) accepted[b] = taken;
  for (uint64_t i = lane; i <= d.drafted; i += kWave) {
    out[b * (size_t(d.drafted) + 1u) + i] = i < taken ? d.token[b * d.drafted + i] : i == taken ? drawn : kNoClass;
  }
}

// One workgroup a sequence: its waves sum the row's blocks in turn, the first of them draws the token.  Bound by the chain of
// loads -- token, its probabilities, the row, then block, groups and class of what is drawn -- 9.6 us for 200 sequences of
// 32768 classes, whose rows alone take 4.
template <int THREADS, int NT>
__global__ __launch_bounds__(THREADS) void verify_kernel(Drafts d, uint32_t sequences, uint32_t blocks,
                                                         const float *__restrict__ pick, uint32_t *__restrict__ out,
                                                         uint32_t *__restrict__ accepted) {
  __shared__ BlockSum sums[kMostHeld];
  const RowGroups<float> rg(d.n);
  for (size_t b = blockIdx.x; b < sequences; b += gridDim.x) {
    uint32_t length;
    const uint32_t taken = taken_tokens(d, b, length);
    const Weights ws = weights_of(d, b, taken, taken < length);
    for (uint32_t i = threadIdx.x / kWave; i < blocks; i += THREADS / kWave) {
      const BlockSum s = ws.q != nullptr ? sum_block<true, NT>(rg, ws, i * kBlockGroups) : sum_block<false, NT>(rg, ws, i * kBlockGroups);
      if ((threadIdx.x & (kWave - 1)) == 0) sums[i] = s;
    }
    __syncthreads();
    if (threadIdx.x < uint32_t(kWave)) {
      write_tokens(d, b, taken, draw_token(rg, ws, blocks, sums, double(pick[b])), out, accepted);
    }
    __syncthreads();
  }
}

// What the summing kernel leaves for the drawing kernel.
struct Sums {
  BlockSum *block;   // [blocks, sequences]
  uint32_t *taken;   // [sequences]: tokens taken, and the top bit where one was refused
};
constexpr uint32_t kRefused = 0x80000000u;

// One wave a block of a sequence's row (every wave finds out for itself which row that is).  Bound by reading: 1024 sequences of
// 131072 classes, half of them with a refusal, 128 us (6.5 TB/s).  64-bit sums are free there: a wave waits 72 % of its time.
template <int NT>
__global__ __launch_bounds__(kDrawThreads) void draw_sums_kernel(Drafts d, uint32_t sequences, uint32_t blocks, Sums out) {
  const RowGroups<float> rg(d.n);
  const uint64_t items = uint64_t(sequences) * blocks;
  for (uint64_t item = uint64_t(blockIdx.x) * kDrawWaves + threadIdx.x / kWave; item < items;
       item += uint64_t(gridDim.x) * kDrawWaves) {
    const size_t b = item / blocks;
    const uint32_t i = uint32_t(item % blocks);
    uint32_t length;
    const uint32_t taken = taken_tokens(d, b, length);
    const bool refused = taken < length;
    const bool lead = (threadIdx.x & (kWave - 1)) == 0;
    if (i == 0u && lead) out.taken[b] = taken | (refused ? kRefused : 0u);
    const Weights ws = weights_of(d, b, taken, refused);
    const BlockSum s = ws.q != nullptr ? sum_block<true, NT>(rg, ws, i * kBlockGroups) : sum_block<false, NT>(rg, ws, i * kBlockGroups);
    if (lead) out.block[item] = s;
  }
}

// One wave a sequence.  A chain of four loads: 3.3 us for one sequence, 8 for 1024.
__global__ __launch_bounds__(kWave) void draw_kernel(Drafts d, uint32_t sequences, uint32_t blocks, Sums in,
                                                     const float *__restrict__ pick, uint32_t *__restrict__ out,
                                                     uint32_t *__restrict__ accepted) {
  const RowGroups<float> rg(d.n);
  for (size_t b = blockIdx.x; b < sequences; b += gridDim.x) {
    const uint32_t word = in.taken[b], taken = word & ~kRefused;
    const Weights ws = weights_of(d, b, taken, (word & kRefused) != 0u);
    write_tokens(d, b, taken, draw_token(rg, ws, blocks, in.block + b * blocks, double(pick[b])), out, accepted);
  }
}

// Blocks of a row, one at least.
uint32_t blocks_of(uint32_t n) {
  const uint32_t groups = n / 4u + (n % 4u != 0u);
  return groups == 0u ? 1u : groups / kBlockGroups + (groups % kBlockGroups != 0u);
}

}  // namespace

size_t verify_scratch(uint32_t classes, uint32_t sequences) {
  const uint32_t blocks = blocks_of(classes);
  return blocks <= kMostHeld ? 0u : size_t(sequences) * (blocks * sizeof(BlockSum) + sizeof(uint32_t));
}
}  // namespace anode

// The most that any of the entry points over rows of classes asks of the stream's scratch.
ANODE_EXPORT size_t anode_gpu_class_rows_scratch_bytes(uint32_t dim0, uint32_t dim1, uint32_t k) {
  size_t most = anode::distill_scratch(dim0, dim1);
  const size_t top = anode::top_k_scratch(dim0, dim1, k), verify = anode::verify_scratch(dim0, dim1);
  if (top > most) most = top;
  return verify > most ? verify : most;
}

ANODE_EXPORT int anode_gpu_verify_draft_packed_f32(uint32_t dim0, uint32_t dim1, uint32_t dim2, const float *target,
                                                   const float *draft, const uint32_t *draft_token, const uint32_t *draft_length,
                                                   const float *accept, const float *pick, uint32_t *token, uint32_t *accepted,
                                                   const KernelConfig *, CUstream_st *stream) {
  using namespace anode;
  const char *const symbol = __func__;
  if (dim2 == 0u) return 0;
  if (dim0 != 0u && target == nullptr) return refuse(symbol, "the target's probabilities are missing");
  if (dim1 != 0u && (draft_token == nullptr || accept == nullptr)) return refuse(symbol, "the drafted tokens are missing");
  if (pick == nullptr || token == nullptr || accepted == nullptr) return refuse(symbol, "an array is missing");
  if (dim1 >= kRefused) return refuse(symbol, "more drafted tokens than 2^31 - 1");
  const hipStream_t st = as_stream(stream);
  const uint32_t blocks = blocks_of(dim0);
  const Drafts d = {dim0, dim1, target, draft, draft_token, draft_length, accept};
  // a token's rows are read once, past the caches where they are large (the model's other rows are not read at all)
  const bool nt = (stream_policy(size_t(dim2) * dim0 * 2u * sizeof(float), tuning().reduce_nontemporal) & kNtLoad) != 0;
  const uint32_t cus = uint32_t(device_cu_count());
  if (blocks <= kMostHeld) {
    // one launch, a workgroup a sequence, as wide as lets all of them run at once
    auto go = [&](auto *kernel, uint32_t threads) {
      return note_launched(symbol, launch(kernel, dim2, threads, 0, st, d, dim2, blocks, pick, token, accepted));
    };
    if (blocks <= 4u || dim2 > 2u * cus) return nt ? go(&verify_kernel<256, kNtLoad>, 256u) : go(&verify_kernel<256, 0>, 256u);
    if (dim2 > cus) return nt ? go(&verify_kernel<512, kNtLoad>, 512u) : go(&verify_kernel<512, 0>, 512u);
    return nt ? go(&verify_kernel<1024, kNtLoad>, 1024u) : go(&verify_kernel<1024, 0>, 1024u);
  }
  const RowsScratch scratch = rows_scratch(st, verify_scratch(dim0, dim2), symbol);
  if (scratch.error != 0) return scratch.error;
  char *at = static_cast<char *>(scratch.lease.ptr);
  const Sums sums = {reinterpret_cast<BlockSum *>(at), reinterpret_cast<uint32_t *>(at + size_t(dim2) * blocks * sizeof(BlockSum))};
  const uint64_t items = (uint64_t(dim2) * blocks + kDrawWaves - 1u) / kDrawWaves;
  const hipError_t e = launch(nt ? &draw_sums_kernel<kNtLoad> : &draw_sums_kernel<0>, items, kDrawThreads, 0,
                              st, d, dim2, blocks, sums);
  if (e != hipSuccess) return note_launched(symbol, e);
  return note_launched(symbol, launch(&draw_kernel, dim2, kWave, 0, st, d, dim2, blocks, sums, pick, token, accepted));
}
