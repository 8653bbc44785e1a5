// Verification of drafted tokens (akh_verify_drafts): speculative sampling's
// acceptance rule on the target's and the draft's logits.
//
// A row's probabilities are e^((l - max) / T) / sum in f64, as the sampler's
// are.  Three launches: k_verify_stats reduces every row in parts of kPart
// ids (maximum, its first index, the sum relative to the part's maximum);
// k_verify_rest, a block per sequence and part, joins the parts of the
// sequence's rows, finds its first refused draft and sums the weights of the
// last token's distribution in chunks of 64 ids; k_verify_pick scans those sums for
// the chunk, and the chunk for the id, where the cumulative weight passes the
// draw.
#include <hip/hip_runtime.h>

#include "common.h"
#include "kernels.h"

namespace akh {

namespace {

constexpr int kPart = 4096;        // ids of a row that one block takes
constexpr int kPer = kPart / 256;  // of them a thread's
constexpr int kChunk = 64;         // ids whose weights k_verify_rest sums together
constexpr int kChunks = kPart / kChunk;

struct PartStat {
  double sum;      // of 2^(c (l - max)), c = log2(e) / T
  float max;       // -infinity: no number in the part
  uint32_t first;  // its first index
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
  uint32_t pad;
};

template <int CTRL>
__device__ __forceinline__ double dpp_f64(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_mov_dpp((int)(uint32_t)u, CTRL, 0xF, 0xF, true);
  const uint32_t hi = __builtin_amdgcn_mov_dpp((int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Sum over aligned groups of 16 lanes (the partners of group_sum), over the
// wave, over the block of 256; every lane gets it.
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
__device__ __forceinline__ double block_sum_f64(double v, double* red4) {
  v = wave_sum_f64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red4[threadIdx.x >> 6] = v;
  __syncthreads();
  return ((red4[0] + red4[1]) + red4[2]) + red4[3];
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

// Weight 2^(c (l - max)) of a logit next to its row's (or part's) maximum: a
// power of two and the Taylor polynomial of 2^f, |f| <= 1/2, whose degree 10
// leaves 2e-13.  The whole part n comes from the low bits of t + 1.5 2^52 and goes
// into the exponent field as an integer, so that but for one conversion every
// step is a full-rate f64 operation (weights below 2^-1000 are left out; that is far under the
// sums' last bit).  A NaN, and an infinity next to an infinite maximum, has none.
__device__ __forceinline__ double weight(float l, float max, double c) {
  const double d = (double)l - (double)max;
  const double m = fma(d, c, 0x1.8p52);
  const double f = fma(d, c, -(m - 0x1.8p52));
  double p = 7.05491162080112088e-09;
  p = fma(p, f, 1.01780860092396960e-07);
  p = fma(p, f, 1.32154867901443053e-06);
  p = fma(p, f, 1.52527338040598377e-05);
  p = fma(p, f, 1.54035303933816061e-04);
  p = fma(p, f, 1.33335581464284411e-03);
  p = fma(p, f, 9.61812910762847688e-03);
  p = fma(p, f, 5.55041086648215762e-02);
  p = fma(p, f, 2.40226506959100694e-01);
  p = fma(p, f, 6.93147180559945286e-01);
  p = fma(p, f, 1.0);
  const uint64_t u = __builtin_bit_cast(uint64_t, p);
  const uint32_t hi = (uint32_t)(u >> 32) + ((uint32_t)__builtin_bit_cast(uint64_t, m) << 20);
  const double w = __builtin_bit_cast(double, (uint64_t)hi << 32 | (uint32_t)u);
  return m > 0x1.8p52 - 1000.0 ? w : 0.0;
}

__device__ __forceinline__ double log2_scale(float temperature) {
  return 1.4426950408889634 / (double)temperature;
}

__device__ __forceinline__ uint32_t drafts_of(const VerifyArgs& a, uint32_t b) {
  return a.counts ? min(a.counts[b], a.rows) : a.rows;
}

// Rows of target first, then of draft.
__global__ __launch_bounds__(256) void k_verify_stats(VerifyArgs a, PartStat* stats, int parts) {
  const uint64_t row = blockIdx.x / parts;
  const int part = blockIdx.x % parts;
  const uint64_t trows = (uint64_t)a.batch * (a.rows + 1);
  const bool is_target = row < trows;
  const uint64_t r = is_target ? row : row - trows;
  const uint32_t per = is_target ? a.rows + 1 : a.rows;
  const uint32_t b = (uint32_t)(r / per), t = (uint32_t)(r % per);
  const uint32_t c = drafts_of(a, b);
  if (is_target ? t > c : t >= c) return;
  const float* l = (is_target ? a.target : a.draft) + r * a.n;
  float x[kPer];
  const uint32_t id0 = part * kPart + threadIdx.x;
#pragma unroll
  for (int i = 0; i < kPer; ++i) x[i] = l[min(id0 + i * 256, a.n - 1)];
#pragma unroll
  for (int i = 0; i < kPer; ++i) x[i] = id0 + i * 256 < a.n ? x[i] : NAN;
  float best = -INFINITY;
  uint32_t first = 0xFFFFFFFFu;
#pragma unroll
  for (int i = kPer - 1; i >= 0; --i)
    if (x[i] >= best) {
      best = x[i];
      first = id0 + i * 256;
    }
  block_amax256(best, first);
  double sum = 0.0;
  if (a.temperature > 0.f) {
    const double c2 = log2_scale(a.temperature);
    __shared__ double red[4];
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum += weight(x[i], best, c2);
    sum = block_sum_f64(sum, red);
  }
  if (threadIdx.x == 0) stats[blockIdx.x] = {sum, best, first};
}

// Joins a row's parts, 16 lanes to a row (all of them get it); mine: the
// lane's own part, or one without a number.
__device__ __forceinline__ PartStat own_part(const PartStat* s, int parts, int lane) {
  return s[min(lane, parts - 1)];
}
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

// What an id's weight for the last token is made of: its logits.
struct IdLogits {
  float p, q;  // q: 1 or 0 for drafts without logits
};
__device__ __forceinline__ IdLogits id_logits(const VerifyArgs& a, const Decision& d, uint32_t b,
                                              uint32_t id, bool less_q) {
  const uint32_t at = min(id, a.n - 1);
  const size_t row = (size_t)b * a.rows + d.row;
  IdLogits x{a.target[(row + b) * a.n + at], 0.f};
  if (less_q) x.q = a.draft ? a.draft[row * a.n + at] : (d.token == id ? 1.f : 0.f);
  if (id >= a.n) x.p = NAN;
  return x;
}
// p, less q where a draft was refused; nothing past the row's end.
__device__ __forceinline__ double id_weight(const VerifyArgs& a, const Decision& d, IdLogits x,
                                            double c, double inv_p, double inv_q, bool less_q) {
  const double p = weight(x.p, d.p.max, c) * inv_p;
  if (!less_q) return p;
  const double q = a.draft ? weight(x.q, d.q.max, c) * inv_q : (double)x.q;
  return fmax(p - q, 0.0);
}
__device__ __forceinline__ double inverse(double x) { return x > 0.0 ? 1.0 / x : 0.0; }

// A block per sequence and part (one part when greedy).  Every block joins
// the sequence's rows, 16 at a time with 16 lanes each, up to the first refused draft.
__global__ __launch_bounds__(256) void k_verify_rest(VerifyArgs a, const PartStat* stats,
                                                     double* sums, Decision* decisions,
                                                     int parts) {
  const bool greedy = !(a.temperature > 0.f);
  const int per = greedy ? 1 : parts;  // blocks of a sequence: no weights to sum when greedy
  const uint32_t b = blockIdx.x / per;
  const int part = blockIdx.x % per;
  const uint32_t c = drafts_of(a, b);
  const double c2 = greedy ? 1.0 : log2_scale(a.temperature);
  const uint64_t trow = (uint64_t)b * (a.rows + 1);
  const uint64_t qrow = (uint64_t)a.batch * (a.rows + 1) + (uint64_t)b * a.rows;
  const int group = threadIdx.x >> 4, lane16 = threadIdx.x & 15;
  __shared__ uint32_t refused;
  __shared__ Decision dec;
  if (threadIdx.x == 0) refused = c;
  bool decided = false;
  // Past the refused row only the chances are wanted, of the first part's block.
  for (uint32_t t0 = 0; t0 <= c; t0 += 16) {
    const uint32_t t = t0 + group;
    // Loaded whether or not the row is live (inside the buffers either way), so that
    // counts, tokens and the parts arrive together.
    const uint32_t tr = min(t, a.rows), td = min(t, a.rows ? a.rows - 1 : 0);
    const uint32_t x = a.rows ? a.tokens[(size_t)b * a.rows + td] : 0u;
    const PartStat* sp = stats + (trow + tr) * parts;
    const PartStat* sq = stats + (qrow + td) * parts;
    const PartStat mp = own_part(sp, parts, lane16);
    const bool two = a.draft != nullptr;
    const PartStat mq = two ? own_part(sq, parts, lane16) : PartStat{0.0, -INFINITY, 0};
    const double u = greedy ? 0.0 : a.uniforms[(size_t)b * (a.rows + 1) + tr];
    const uint32_t xi = x < a.n ? x : 0;
    const float lp = a.target[(trow + tr) * a.n + xi];
    const float lq = two ? a.draft[((size_t)b * a.rows + td) * a.n + xi] : 0.f;
    RowStat p{}, q{};
    bool ok = true;
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
    if (!decided && refused < t0 + 16) {
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
  }
  __syncthreads();
  if (part == 0) {
    const uint32_t r = dec.row;
    for (uint32_t t = threadIdx.x; t <= a.rows; t += 256) {
      if (t != r) a.out_tokens[trow + t] = t < r ? a.tokens[(size_t)b * a.rows + t] : 0xFFFFFFFFu;
      if (t >= c && t < a.rows && a.chance) a.chance[(size_t)b * a.rows + t] = 0.f;
    }
    if (threadIdx.x == 0) {
      a.out_counts[b] = r + 1;
      if (greedy) a.out_tokens[trow + r] = dec.p.first;
      decisions[b] = dec;
    }
  }
  if (greedy) return;
  const Decision d = dec;
  const double inv_p = inverse(d.p.sum), inv_q = inverse(d.q.sum);
  const int wave = threadIdx.x >> 6;
  double* s = sums + ((size_t)b * parts + part) * kChunks;
  IdLogits x[kPer];
  const uint32_t id0 = part * kPart + threadIdx.x;
#pragma unroll
  for (int i = 0; i < kPer; ++i) x[i] = id_logits(a, d, b, id0 + i * 256, d.has_q);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const double w = wave_sum_f64(id_weight(a, d, x[i], c2, inv_p, inv_q, d.has_q));
    if ((threadIdx.x & 63) == 0) s[i * 4 + wave] = w;
  }
}

// A block per sequence: the chunk of ids in which the cumulative weight
// passes the draw, then the id in it.
__global__ __launch_bounds__(256) void k_verify_pick(VerifyArgs a, double* sums,
                                                     const Decision* decisions, int parts) {
  const uint32_t b = blockIdx.x;
  const Decision d = decisions[b];
  const double c2 = log2_scale(a.temperature);
  const double inv_p = inverse(d.p.sum), inv_q = inverse(d.q.sum);
  const double u = a.uniforms[(size_t)b * (a.rows + 1) + a.rows];
  uint32_t* out = a.out_tokens + (size_t)b * (a.rows + 1) + d.row;
  double* s = sums + (size_t)b * parts * kChunks;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = parts * kChunks, per = n / 256 + (n % 256 != 0);
  const int i0 = min(n, (int)threadIdx.x * per), i1 = min(n, i0 + per);
  __shared__ double tot[4];
  __shared__ int hit, last;
  __shared__ double base;
  bool less_q = d.has_q;
  double before = 0.0, total = 0.0;
  for (int round = 0; round < 2; ++round) {
    double own = 0.0;
    for (int i = i0; i < i1; ++i) own += s[i];
    const double upto = wave_scan_f64(own, lane);
    if (lane == 63) tot[wave] = upto;
    if (threadIdx.x == 0) {
      hit = n;
      last = -1;
    }
    __syncthreads();
    before = upto - own;
    for (int w = 0; w < wave; ++w) before += tot[w];
    total = ((tot[0] + tot[1]) + tot[2]) + tot[3];
    if (total > 0.0 || !less_q) break;
    // Nothing of p exceeds q: p itself, whose sums are made here.
    less_q = false;
    for (int i = threadIdx.x; i < n; i += 256) {
      double w = 0.0;
      for (int k = 0; k < kChunk; ++k) {
        const uint32_t id = (uint32_t)i * kChunk + k;
        w += id_weight(a, d, id_logits(a, d, b, id, false), c2, inv_p, inv_q, false);
      }
      s[i] = w;
    }
    __syncthreads();
  }
  if (!(total > 0.0)) {
    if (threadIdx.x == 0) *out = d.p.first;
    return;
  }
  const double point = u * total;
  double cum = before;
  int mine = n, weighty = -1;
  for (int i = i0; i < i1; ++i) {
    const double w = s[i];
    cum += w;
    if (w > 0.0) {
      weighty = i;
      if (cum > point && mine == n) mine = i;
    }
  }
  if (mine < n) atomicMin(&hit, mine);
  if (weighty >= 0) atomicMax(&last, weighty);
  __syncthreads();
  const int chunk = hit < n ? hit : last;  // rounding may leave none past the point
  if (chunk >= i0 && chunk < i1) {
    cum = before;
    for (int i = i0; i < chunk; ++i) cum += s[i];
    base = cum;
  }
  __syncthreads();
  if (wave) return;
  const uint32_t id = (uint32_t)chunk * kChunk + lane;
  const double w = id_weight(a, d, id_logits(a, d, b, id, less_q), c2, inv_p, inv_q, less_q);
  const double upto = base + wave_scan_f64(w, lane);
  const uint64_t some = __ballot(w > 0.0), past = __ballot(w > 0.0 && upto > point);
  const int k = past ? __ffsll((unsigned long long)past) - 1 : 63 - __clzll((long long)some);
  if (lane == 0) *out = (uint32_t)chunk * kChunk + k;
}

int parts_of(uint32_t n) { return (int)((n + kPart - 1) / kPart); }
uint64_t stat_rows(uint32_t batch, uint32_t rows) { return (uint64_t)batch * (2 * (uint64_t)rows + 1); }

}  // namespace

uint64_t verify_blocks(uint32_t batch, uint32_t rows, uint32_t n) {
  return stat_rows(batch, rows) * parts_of(n);
}

size_t verify_workspace_bytes(uint32_t batch, uint32_t rows, uint32_t n) {
  return verify_blocks(batch, rows, n) * sizeof(PartStat) +
         (size_t)batch * (parts_of(n) * kChunks * sizeof(double) + sizeof(Decision));
}

hipError_t launch_verify(const VerifyArgs& a, hipStream_t s) {
  const int parts = parts_of(a.n);
  PartStat* stats = static_cast<PartStat*>(a.ws);
  double* sums = reinterpret_cast<double*>(stats + verify_blocks(a.batch, a.rows, a.n));
  Decision* dec = reinterpret_cast<Decision*>(sums + (size_t)a.batch * parts * kChunks);
  const uint64_t rows = a.draft ? stat_rows(a.batch, a.rows) : (uint64_t)a.batch * (a.rows + 1);
  hipLaunchKernelGGL(k_verify_stats, dim3((uint32_t)(rows * parts)), dim3(256), 0, s, a, stats,
                     parts);
  hipLaunchKernelGGL(k_verify_rest, dim3((uint32_t)(a.temperature > 0.f ? a.batch * parts : a.batch)),
                     dim3(256), 0, s, a, stats, sums, dec, parts);
  if (a.temperature > 0.f)
    hipLaunchKernelGGL(k_verify_pick, dim3(a.batch), dim3(256), 0, s, a, sums, dec, parts);
  return hipGetLastError();
}

}  // namespace akh
