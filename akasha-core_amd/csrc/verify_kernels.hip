// Verification of drafted tokens (akh_verify_drafts): speculative sampling's
// acceptance rule on the target's and the draft's logits.
//
// A row's probabilities are e^((l - max) / T) / sum in f64, as the sampler's
// are.  Two launches.  k_verify_stats reduces every row in parts of kPart
// ids: maximum, and the sum of weights relative to the part's maximum.  Then a
// block per sequence and part (k_verify_pick) joins the parts of the sequence's rows, finds its
// first refused draft and sums its part's weights of the last token's
// distribution in chunks of 16 ids; the sequence's last block to finish walks
// the parts' sums, the chunks' and the chunk's ids to the one where the
// cumulative weight passes the draw.
#include <hip/hip_runtime.h>

#include "common.h"
#include "kernels.h"

namespace akh {

namespace {

constexpr int kPart = 4096;          // ids of a row that one block takes
constexpr int kPer = kPart / 256;    // of them a thread's, for the statistics
constexpr int kPick = 256;           // threads of a block for the last token
constexpr int kChunk = kPart / kPick;  // ids of one of them, in a row
constexpr int kWaves = kPick / 64;
constexpr int kPreload = 16;         // parts whose chunk sums are fetched before one is chosen

struct PartStat {
  double sum;      // of 2^(c (l - max)), c = log2(e) / T
  float max;       // -infinity: no number in the part
  uint32_t first;  // its first index, for greedy calls
};
struct RowStat {
  double sum;
  float max;
  uint32_t first;
};
// What a sequence's last token is drawn from.
struct Decision {
  RowStat p, q;
  uint32_t row;    // of the target
  uint32_t has_q;  // a draft was refused there,
  uint32_t token;  // this one
};

template <int CTRL>
__device__ __forceinline__ double dpp_f64(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_mov_dpp((int)(uint32_t)u, CTRL, 0xF, 0xF, true);
  const uint32_t hi = __builtin_amdgcn_mov_dpp((int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Sum over aligned groups of 16 lanes (the partners of group_sum), over the
// wave, over the block; every lane gets it.
__device__ __forceinline__ double sum16_f64(double v) {
  v += dpp_f64<0xB1>(v);
  v += dpp_f64<0x4E>(v);
  v += dpp_f64<0x141>(v);
  v += dpp_f64<0x140>(v);
  return v;
}
// x[lane] + x[lane ^ O], O = 16 or 32, as xor_sum: the swaps leave both halves
// of the pair's numbers in the same order.
template <int O>
__device__ __forceinline__ double xor_sum_f64(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)u, hi = (uint32_t)(u >> 32);
  uint64_t a, b;
  if constexpr (O == 16) {
    const auto l = __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
    const auto h = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
    a = (uint64_t)h[0] << 32 | l[0];
    b = (uint64_t)h[1] << 32 | l[1];
  } else {
    const auto l = __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
    const auto h = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
    a = (uint64_t)h[0] << 32 | l[0];
    b = (uint64_t)h[1] << 32 | l[1];
  }
  return __builtin_bit_cast(double, a) + __builtin_bit_cast(double, b);
}
__device__ __forceinline__ double wave_sum_f64(double v) {
  return xor_sum_f64<32>(xor_sum_f64<16>(sum16_f64(v)));
}
template <int WAVES>
__device__ __forceinline__ double block_sum_f64(double v, double* red) {
  v = wave_sum_f64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int i = 1; i < WAVES; ++i) v += red[i];
  return v;
}
// Sum over the wave's lanes up to and with this one.
__device__ __forceinline__ double wave_scan_f64(double v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}
// Where a walk over the block's weights passes `point`, starting at `base`:
// the thread, and what lies before it.  Rounding may leave none past the
// point: the last one with weight then.
struct Step {
  int at;
  double before;
};
struct StepShared {
  double tot[kWaves];
  Step hit[kWaves], last[kWaves];  // of each wave; at < 0: none
};
__device__ Step walk(double w, double base, double point, StepShared& sh) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const double upto = wave_scan_f64(w, lane);
  if (lane == 63) sh.tot[wave] = upto;
  __syncthreads();
  double before = base + (upto - w);
  for (int i = 0; i < wave; ++i) before += sh.tot[i];
  const uint64_t some = __ballot(w > 0.0);
  const uint64_t past = __ballot(w > 0.0 && before + w > point);
  const int hit = past ? __builtin_ctzll(past) : -1;
  const int last = some ? 63 - __builtin_clzll(some) : -1;
  const int id = threadIdx.x;
  if (lane == (hit < 0 ? 0 : hit)) sh.hit[wave] = {hit < 0 ? -1 : id, before};
  if (lane == (last < 0 ? 0 : last)) sh.last[wave] = {last < 0 ? -1 : id, before};
  __syncthreads();
  Step at = {0, base};
#pragma unroll
  for (int i = 0; i < kWaves; ++i)
    if (sh.last[i].at >= 0) at = sh.last[i];
#pragma unroll
  for (int i = kWaves - 1; i >= 0; --i)
    if (sh.hit[i].at >= 0) at = sh.hit[i];
  return at;
}

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
// 2^(n + f) from m = 1.5 2^52 + n and |f| <= 1/2: the polynomial that agrees
// with 2^f in the ten Chebyshev points of [-1/2, 1/2] (within 4e-14 of it, and
// 1 at 0), times 2^n, n being m's low half as an integer.
__device__ __forceinline__ double power2(double m, double f) {
  double p = 0x1.b6571de2f2351p-24;
  p = fma(p, f, 0x1.63ef969a64d3cp-20);
  p = fma(p, f, 0x1.ffcb76789860fp-17);
  p = fma(p, f, 0x1.43088e257f341p-13);
  p = fma(p, f, 0x1.5d87fe908f88ap-10);
  p = fma(p, f, 0x1.3b2ab72b175eep-7);
  p = fma(p, f, 0x1.c6b08d7044119p-5);
  p = fma(p, f, 0x1.ebfbdff8149f2p-3);
  p = fma(p, f, 0x1.62e42fefa39f7p-1);
  p = fma(p, f, 1.0);
  return ldexp(p, (int)__builtin_bit_cast(u32x2, m).x);
}
// Weight 2^(c (l - max)) of a logit next to its row's (or part's) maximum; none
// for a NaN, and for an infinity next to an infinite maximum.  (Weights below
// 2^-1000 are left out, far under the sums' last bit.)
__device__ __forceinline__ double weight(float l, float max, double c) {
  const double d = (double)l - (double)max;
  const double m = fma(d, c, 0x1.8p52);
  const double w = power2(m, fma(d, c, -(m - 0x1.8p52)));
  return m > 0x1.8p52 - 1000.0 ? w : 0.0;
}
// The same for a sum next to which 2^-1000 is nothing: least = -1000 / c.
__device__ __forceinline__ double weight_in_sum(float l, float max, double c, double least) {
  const double d = fmax((double)l - (double)max, least);
  const double m = fma(d, c, 0x1.8p52);
  return power2(m, fma(d, c, -(m - 0x1.8p52)));
}

// Not 0 for an infinite temperature, whose weights of -infinity stay none.
__device__ __forceinline__ double log2_scale(float temperature) {
  return fmax(1.4426950408889634 / (double)temperature, 1e-60);
}

__device__ __forceinline__ uint32_t drafts_of(const VerifyArgs& a, uint32_t b) {
  return a.counts ? min(a.counts[b], a.rows) : a.rows;
}

// A thread's ids of a part, 256 apart; NaN past the row's end.
__device__ __forceinline__ void load_part(const float* row, uint32_t n, int part, float* x) {
  const uint32_t here = min(n - (uint32_t)part * kPart, (uint32_t)kPart);
  const float* p = row + (size_t)part * kPart;
  if (here == kPart) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = p[i * 256 + threadIdx.x];
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = p[min(i * 256 + threadIdx.x, here - 1)];
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i * 256 + threadIdx.x >= here) x[i] = NAN;
  }
}

// Rows of target first, then of draft.  32 sequences of 0 to 7 drafts over
// 50257 ids, 256 rows live (51 MB), take 16 us, 3.1 TB/s, where a sum over 1 GB
// reads at 4.1: the f64 arithmetic, 20 instructions an id, is half of that
// long and the reads' start and end are seen.  (40 instructions, with the first
// maximum's index kept in every call, compares and 64-bit exponent sums: 22
// us; parts of 2048 ids 20 us; a sum next to each wave's own maximum the same.)
__global__ __launch_bounds__(256) void k_verify_stats(VerifyArgs a, PartStat* stats, int* done,
                                                      int parts) {
  const uint32_t row = blockIdx.x / parts;
  const int part = blockIdx.x - row * parts;
  const uint32_t trows = a.batch * (a.rows + 1);
  const bool is_target = row < trows;
  const uint32_t r = is_target ? row : row - trows;
  const uint32_t per = is_target ? a.rows + 1 : a.rows;
  const uint32_t b = r / per, t = r - b * per;
  if (is_target && t == 0 && part == 0 && threadIdx.x == 0) done[b] = 0;  // for k_verify_pick
  const uint32_t c = drafts_of(a, b);
  if (is_target ? t > c : t >= c) return;
  float x[kPer];
  load_part((is_target ? a.target : a.draft) + (size_t)r * a.n, a.n, part, x);
  if (!(a.temperature > 0.f)) {
    float best = -INFINITY;
    uint32_t first = 0xFFFFFFFFu;
#pragma unroll
    for (int i = kPer - 1; i >= 0; --i)
      if (x[i] >= best) {
        best = x[i];
        first = part * kPart + i * 256 + threadIdx.x;
      }
    block_amax256(best, first);
    if (threadIdx.x == 0) stats[blockIdx.x] = {0.0, best, first};
    return;
  }
  __shared__ float red_f[4];
  __shared__ double red_d[4];
  float best = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPer; ++i) best = fmaxf(best, x[i]);
  best = block_max256(best, red_f);
  const double c2 = log2_scale(a.temperature), least = -1000.0 / c2;
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) sum += weight_in_sum(x[i], best, c2, least);
  sum = block_sum_f64<4>(sum, red_d);
  if (threadIdx.x == 0)
    stats[blockIdx.x] = {fabsf(best) < INFINITY ? sum : 0.0, best, 0xFFFFFFFFu};
}

__device__ __forceinline__ PartStat own_part(const PartStat* s, int parts, int lane) {
  return s[min(lane, parts - 1)];
}
// Joins a row's parts, 16 lanes to a row (all of them get it); mine: the
// lane's first part.
__device__ __forceinline__ RowStat join16(const PartStat* s, PartStat mine, int parts, double c,
                                          int lane) {
  if (lane >= parts) mine = {0.0, -INFINITY, 0xFFFFFFFFu};
  float m = mine.max;
  uint32_t first = mine.first;
  for (int i = lane + 16; i < parts; i += 16)
    if (s[i].max > m || (s[i].max == m && s[i].first < first)) {
      m = s[i].max;
      first = s[i].first;
    }
  const float top = group_max<16>(m);
  first = m == top ? first : 0xFFFFFFFFu;
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) first = min(first, (uint32_t)__shfl_xor((int)first, o, 64));
  double z = mine.sum * weight(mine.max, top, c);
  for (int i = lane + 16; i < parts; i += 16) z += s[i].sum * weight(s[i].max, top, c);
  return {sum16_f64(z), top, first == 0xFFFFFFFFu ? 0u : first};
}

__device__ __forceinline__ double prob(float l, const RowStat& s, double c) {
  return s.sum > 0.0 ? weight(l, s.max, c) / s.sum : 0.0;
}

// What an id's weight for the last token is made of.
struct Draw {
  const float* p;  // the target's row
  const float* q;  // the draft's, or null
  uint32_t token;  // the draft without a distribution, or no id
  float pm, qm;
  double c, inv_p, inv_q;
  bool less_q;

  // q without logits: 1 or 0.
  __device__ __forceinline__ double of(float lp, float lq) const {
    const double w = weight(lp, pm, c) * inv_p;
    if (!less_q) return w;
    return fmax(w - (q ? weight(lq, qm, c) * inv_q : (double)lq), 0.0);
  }
  __device__ __forceinline__ double of_id(uint32_t id, uint32_t n) const {
    if (id >= n) return 0.0;
    return of(p[id], !less_q ? 0.f : q ? q[id] : token == id ? 1.f : 0.f);
  }
};

__device__ __forceinline__ double agent_load(const double* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void agent_store(double* p, double x) {
  __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// A thread's kChunk ids in a row of a part; NaN past the row's end.
__device__ __forceinline__ void load_chunk(const float* row, uint32_t n, int part, float* x) {
  typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
  const uint32_t here = min(n - (uint32_t)part * kPart, (uint32_t)kPart);
  const float* p = row + (size_t)part * kPart;
  const uint32_t at = threadIdx.x * kChunk;
  if (here == kPart) {
#pragma unroll
    for (int i = 0; i < kChunk; i += 4) {
      const f4 v = *reinterpret_cast<const f4*>(p + at + i);
#pragma unroll
      for (int k = 0; k < 4; ++k) x[i + k] = v[k];
    }
  } else {
#pragma unroll
    for (int i = 0; i < kChunk; ++i) x[i] = p[min(at + i, here - 1)];
#pragma unroll
    for (int i = 0; i < kChunk; ++i)
      if (at + i >= here) x[i] = NAN;
  }
}

// A chain of loads and short scans, each waiting for the one before it: 10 us
// for one sequence, 14 us for 32 (two rows of 50257 ids each, 13 MB). As a
// launch of its own after one that sums the chunks it was 8 us on top of 16; the
// hand-off to the last block costs 1.4.  Blocks of 512 or 1024 threads with
// chunks of 8 or 4 ids: 11.5 and 16 us; the parts' logits by way of LDS 10.9.
// A block per sequence and part (one part when greedy).  Every block joins
// the sequence's rows, 16 at a time with 16 lanes each, up to the first refused draft.
// The sums are written through to device scope and counted there; the count
// starts at zero by k_verify_stats.
__global__ __launch_bounds__(kPick) void k_verify_pick(VerifyArgs a, const PartStat* stats,
                                                     double* sums, double* totals, int* done,
                                                     int parts) {
  const bool greedy = !(a.temperature > 0.f);
  const int per = greedy ? 1 : parts;  // blocks of a sequence: no weights to sum when greedy
  const uint32_t b = blockIdx.x / per;
  const int part = blockIdx.x - b * per;
  const uint32_t c = drafts_of(a, b);
  const double c2 = greedy ? 1.0 : log2_scale(a.temperature);
  const uint64_t trow = (uint64_t)b * (a.rows + 1);
  const uint64_t qrow = (uint64_t)a.batch * (a.rows + 1) + (uint64_t)b * a.rows;
  const int group = threadIdx.x >> 4, lane16 = threadIdx.x & 15;
  const double last_u = greedy ? 0.0 : a.uniforms[trow + a.rows];
  __shared__ uint32_t refused;
  __shared__ Decision dec;
  bool decided = false;
  // Past the refused row only the chances are wanted, of the first part's block.
  uint32_t t0 = 0;
  do {
    const uint32_t t = t0 + group;
    // Loaded whether or not the row is live (inside the buffers either way), so that
    // counts, tokens and the parts arrive together.
    const uint32_t tr = min(t, a.rows), td = min(t, a.rows ? a.rows - 1 : 0);
    const uint32_t x = a.rows ? a.tokens[(size_t)b * a.rows + td] : 0u;
    const PartStat* sp = stats + (trow + tr) * parts;
    const PartStat* sq = stats + (qrow + td) * parts;
    const PartStat mp = own_part(sp, parts, lane16);
    const bool two = a.draft != nullptr && a.rows;
    const PartStat mq = two ? own_part(sq, parts, lane16) : PartStat{0.0, -INFINITY, 0};
    const double u = greedy ? 0.0 : a.uniforms[trow + tr];
    const uint32_t xi = x < a.n ? x : 0;
    const float lp = a.target[(trow + tr) * a.n + xi];
    const float lq = two ? a.draft[((size_t)b * a.rows + td) * a.n + xi] : 0.f;
    RowStat p{}, q{};
    bool ok = true;
    if (t0 == 0 && threadIdx.x == 0) refused = c;
    __syncthreads();
    if (t <= c) {
      p = join16(sp, mp, parts, c2, lane16);
      if (two && t < c) q = join16(sq, mq, parts, c2, lane16);
      if (t < c) {
        double chance = 0.0;
        ok = false;
        if (greedy) {
          ok = x == p.first;
          chance = ok ? 1.0 : 0.0;
        } else if (x < a.n) {
          const double px = prob(lp, p, c2);
          const double qx = two ? prob(lq, q, c2) : 1.0;
          ok = u * qx < px;
          chance = px > 0.0 ? fmin(px / qx, 1.0) : 0.0;
        }
        if (lane16 == 0) {
          if (!ok) atomicMin(&refused, t);
          if (part == 0 && a.chance) a.chance[(size_t)b * a.rows + t] = (float)chance;
        }
      }
    }
    __syncthreads();
    if (!decided && refused < t0 + kPick / 16) {
      if (t == refused && lane16 == 0) {
        dec.p = p;
        dec.q = q;
        dec.row = t;
        dec.has_q = t < c;
        dec.token = x;
      }
      decided = true;
      if (part != 0) break;
    }
    t0 += kPick / 16;
  } while (t0 <= c);
  __syncthreads();
  const Decision d = dec;
  if (part == 0) {
    for (uint32_t t = threadIdx.x; t <= a.rows; t += kPick) {
      if (t != d.row)
        a.out_tokens[trow + t] = t < d.row ? a.tokens[(size_t)b * a.rows + t] : 0xFFFFFFFFu;
      if (t >= c && t < a.rows && a.chance) a.chance[(size_t)b * a.rows + t] = 0.f;
    }
    if (threadIdx.x == 0) {
      a.out_counts[b] = d.row + 1;
      if (greedy) a.out_tokens[trow + d.row] = d.p.first;
    }
  }
  if (greedy) return;

  Draw w;
  w.p = a.target + (trow + d.row) * a.n;
  w.less_q = d.has_q;
  w.q = d.has_q && a.draft ? a.draft + ((size_t)b * a.rows + d.row) * a.n : nullptr;
  w.token = d.token;
  w.pm = d.p.max;
  w.qm = d.q.max;
  w.c = c2;
  w.inv_p = d.p.sum > 0.0 ? 1.0 / d.p.sum : 0.0;
  w.inv_q = d.q.sum > 0.0 ? 1.0 / d.q.sum : 0.0;
  __shared__ double red[kWaves];
  {
    float x[kChunk], y[kChunk] = {};
    load_chunk(w.p, a.n, part, x);
    if (w.q) load_chunk(w.q, a.n, part, y);
    if (w.less_q && !w.q) {
      const uint32_t one = w.token - (part * kPart + threadIdx.x * kChunk);
#pragma unroll
      for (int i = 0; i < kChunk; ++i) y[i] = one == (uint32_t)i ? 1.f : 0.f;
    }
    double own = 0.0;
#pragma unroll
    for (int i = 0; i < kChunk; ++i) own += w.of(x[i], y[i]);
    agent_store(sums + ((size_t)b * parts + part) * kPick + threadIdx.x, own);
    const double total = block_sum_f64<kWaves>(own, red);
    if (threadIdx.x == 0) agent_store(totals + (size_t)b * parts + part, total);
  }
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  __shared__ bool last_block;
  if (threadIdx.x == 0)
    last_block = __hip_atomic_fetch_add(done + b, 1, __ATOMIC_RELAXED,
                                        __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
  __syncthreads();
  if (!last_block) return;

  double* s = sums + (size_t)b * parts * kPick + threadIdx.x;
  uint32_t* out = a.out_tokens + trow + d.row;
  double v[kPreload];
#pragma unroll
  for (int i = 0; i < kPreload; ++i) v[i] = i < parts ? agent_load(s + (size_t)i * kPick) : 0.0;
  double mine = (int)threadIdx.x < parts ? agent_load(totals + (size_t)b * parts + threadIdx.x) : 0.0;
  double total = block_sum_f64<kWaves>(mine, red);
  bool fetched = parts <= kPreload;
  if (!(total > 0.0) && w.less_q) {
    // Nothing of p exceeds q: p itself, whose sums are made here.
    w.less_q = false;
    for (int i = 0; i < parts; ++i) {
      double own = 0.0;
      for (int k = 0; k < kChunk; ++k)
        own += w.of_id((uint32_t)i * kPart + threadIdx.x * kChunk + k, a.n);
      agent_store(s + (size_t)i * kPick, own);
      const double sum = block_sum_f64<kWaves>(own, red);
      if ((int)threadIdx.x == i) mine = sum;
    }
    __builtin_amdgcn_s_waitcnt(0);
    total = block_sum_f64<kWaves>(mine, red);
    fetched = false;
  }
  if (!(total > 0.0)) {  // no weight at all: the row's first maximum
    __syncthreads();
    if (threadIdx.x == 0) refused = a.n;
    __syncthreads();
    for (uint32_t id = threadIdx.x; id < a.n; id += kPick)
      if (w.p[id] == w.pm) {
        atomicMin(&refused, id);
        break;
      }
    __syncthreads();
    if (threadIdx.x == 0) *out = refused < a.n ? refused : 0;
    return;
  }
  __shared__ StepShared sh;
  const double point = last_u * total;
  const Step at = walk(mine, 0.0, point, sh);
  double chunk = 0.0;
  if (fetched) {
#pragma unroll
    for (int i = 0; i < kPreload; ++i) chunk = i == at.at ? v[i] : chunk;
  } else {
    chunk = agent_load(s + (size_t)at.at * kPick);
  }
  const Step in = walk(chunk, at.before, point, sh);
  const uint32_t id0 = (uint32_t)at.at * kPart + in.at * kChunk;
  const Step id = walk(threadIdx.x < kChunk ? w.of_id(id0 + threadIdx.x, a.n) : 0.0, in.before,
                       point, sh);
  if (threadIdx.x == 0) *out = id0 + id.at;
}

static_assert(kMaxSampleVocab / kPart <= kPick, "a thread a part of a row");
int parts_of(uint32_t n) { return (int)((n + kPart - 1) / kPart); }
uint64_t stat_rows(uint32_t batch, uint32_t rows) { return (uint64_t)batch * (2 * (uint64_t)rows + 1); }

}  // namespace

uint64_t verify_blocks(uint32_t batch, uint32_t rows, uint32_t n) {
  return stat_rows(batch, rows) * parts_of(n);
}

size_t verify_workspace_bytes(uint32_t batch, uint32_t rows, uint32_t n) {
  return verify_blocks(batch, rows, n) * sizeof(PartStat) +
         (size_t)batch * (parts_of(n) * (kPick + 1) * sizeof(double) + sizeof(int));
}

hipError_t launch_verify(const VerifyArgs& a, hipStream_t s) {
  const int parts = parts_of(a.n);
  PartStat* stats = static_cast<PartStat*>(a.ws);
  double* sums = reinterpret_cast<double*>(stats + verify_blocks(a.batch, a.rows, a.n));
  double* totals = sums + (size_t)a.batch * parts * kPick;
  int* done = reinterpret_cast<int*>(totals + (size_t)a.batch * parts);
  const uint64_t rows = a.draft ? stat_rows(a.batch, a.rows) : (uint64_t)a.batch * (a.rows + 1);
  hipLaunchKernelGGL(k_verify_stats, dim3((uint32_t)(rows * parts)), dim3(256), 0, s, a, stats,
                     done, parts);
  hipLaunchKernelGGL(k_verify_pick, dim3(a.temperature > 0.f ? a.batch * parts : a.batch),
                     dim3(kPick), 0, s, a, stats, sums, totals, done, parts);
  return hipGetLastError();
}

}  // namespace akh
