// Verification of drafted tokens (akh_verify_drafts): speculative sampling's
// acceptance rule on the target's and the draft's logits.
//
// A row's probabilities are e^((l - max) / T) / sum in f64, as the sampler's
// are.  Three launches: k_verify_stats reduces every row in parts of kPart
// ids (maximum, its first index, the sum relative to the part's maximum);
// k_verify_rest, a block per sequence and part, joins the parts of the
// sequence's rows, finds its first refused draft and sums the part's weights of the last
// token's distribution; k_verify_pick walks those sums to the part and
// the id where the cumulative weight passes the draw.
#include <hip/hip_runtime.h>

#include "common.h"
#include "kernels.h"

namespace akh {

namespace {

constexpr int kPart = 4096;  // ids of a row that one block takes
constexpr int kPer = kPart / 256;

struct PartStat {
  double sum;  // of e^((l - max) / T)
  float max;   // -infinity: no number in the part
  uint32_t first;  // its first index
};
struct RowStat {
  double max, sum;
};
// What a sequence's last token is drawn from.
struct Decision {
  RowStat p, q;
  uint32_t row, has_q, first, pad;
};

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// Sum over 256 threads; every thread gets it.
__device__ __forceinline__ double block_sum_f64(double v, double* red4) {
  v = wave_sum_f64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red4[threadIdx.x >> 6] = v;
  __syncthreads();
  return ((red4[0] + red4[1]) + red4[2]) + red4[3];
}

// Weight of a logit relative to its row's (or part's) maximum; a NaN, and an
// infinity next to an infinite maximum, has none.
__device__ __forceinline__ double weight(float l, double max, double inv_t) {
  const double w = exp(((double)l - max) * inv_t);
  return w > 0.0 ? w : 0.0;
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
  float best = -INFINITY;
  uint32_t first = 0xFFFFFFFFu;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint32_t id = part * kPart + i * 256 + threadIdx.x;
    x[i] = id < a.n ? l[id] : -INFINITY;
    if (x[i] > best || (x[i] == best && id < a.n && id < first)) {
      best = x[i];
      first = id;
    }
  }
  block_amax256(best, first);
  double sum = 0.0;
  if (a.temperature > 0.f) {
    const double inv_t = 1.0 / (double)a.temperature;
    __shared__ double red[4];
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum += weight(x[i], best, inv_t);
    sum = block_sum_f64(sum, red);
  }
  if (threadIdx.x == 0) stats[blockIdx.x] = {sum, best, first};
}

// Joins a row's parts.
__device__ RowStat join(const PartStat* s, int parts, double inv_t, uint32_t* first) {
  float m = -INFINITY;
  uint32_t f = 0xFFFFFFFFu;
  for (int i = 0; i < parts; ++i)
    if (s[i].max > m || (s[i].max == m && s[i].first < f)) {
      m = s[i].max;
      f = s[i].first;
    }
  double z = 0.0;
  for (int i = 0; i < parts; ++i) {
    const double w = s[i].sum * exp(((double)s[i].max - m) * inv_t);
    if (w > 0.0) z += w;
  }
  *first = f == 0xFFFFFFFFu ? 0 : f;
  return {(double)m, z};
}

__device__ __forceinline__ double prob(float l, const RowStat& s, double inv_t) {
  return s.sum > 0.0 ? weight(l, s.max, inv_t) / s.sum : 0.0;
}

// The last token's weights of an id: (max(0, p - q), p).
__device__ __forceinline__ void id_weights(const VerifyArgs& a, const Decision& d, uint32_t b,
                                           uint32_t id, double inv_t, double& rest, double& full) {
  full = prob(a.target[((size_t)b * (a.rows + 1) + d.row) * a.n + id], d.p, inv_t);
  rest = full;
  if (d.has_q) {
    const double q =
        a.draft ? prob(a.draft[((size_t)b * a.rows + d.row) * a.n + id], d.q, inv_t)
                : (a.tokens[(size_t)b * a.rows + d.row] == id ? 1.0 : 0.0);
    rest = fmax(full - q, 0.0);
  }
}

__global__ __launch_bounds__(256) void k_verify_rest(VerifyArgs a, const PartStat* stats,
                                                     double2* rest, Decision* decisions,
                                                     int parts) {
  const bool greedy = !(a.temperature > 0.f);
  const int per = greedy ? 1 : parts;  // blocks of a sequence: no weights to sum when greedy
  const uint32_t b = blockIdx.x / per;
  const int part = blockIdx.x % per;
  const uint32_t c = drafts_of(a, b);
  const double inv_t = greedy ? 1.0 : 1.0 / (double)a.temperature;
  const uint64_t trow = (uint64_t)b * (a.rows + 1);
  const uint64_t qrow = (uint64_t)a.batch * (a.rows + 1) + (uint64_t)b * a.rows;
  __shared__ uint32_t refused;
  __shared__ Decision dec;
  __shared__ double red[4];
  if (threadIdx.x == 0) refused = c;
  __syncthreads();
  for (uint32_t t = threadIdx.x; t < a.rows; t += 256) {
    double chance = 0.0;
    if (t < c) {
      const uint32_t x = a.tokens[(size_t)b * a.rows + t];
      uint32_t first;
      const RowStat p = join(stats + (trow + t) * parts, parts, inv_t, &first);
      bool ok = false;
      if (greedy) {
        ok = x == first;
        chance = ok ? 1.0 : 0.0;
      } else if (x < a.n) {
        const double px = prob(a.target[(trow + t) * a.n + x], p, inv_t);
        double qx = 1.0;
        if (a.draft) {
          const RowStat q = join(stats + (qrow + t) * parts, parts, inv_t, &first);
          qx = prob(a.draft[((size_t)b * a.rows + t) * a.n + x], q, inv_t);
        }
        ok = a.uniforms[(size_t)b * (a.rows + 1) + t] * qx < px;
        chance = px > 0.0 ? fmin(px / qx, 1.0) : 0.0;
      }
      if (!ok) atomicMin(&refused, t);
    }
    if (part == 0 && a.chance) a.chance[(size_t)b * a.rows + t] = (float)chance;
  }
  __syncthreads();
  const uint32_t r = refused;
  if (threadIdx.x == 0) {
    dec.row = r;
    dec.has_q = r < c;
    dec.p = join(stats + (trow + r) * parts, parts, inv_t, &dec.first);
    uint32_t unused;
    dec.q = dec.has_q && a.draft ? join(stats + (qrow + r) * parts, parts, inv_t, &unused)
                                 : RowStat{0.0, 0.0};
    if (part == 0) decisions[b] = dec;
  }
  __syncthreads();
  if (part == 0) {
    for (uint32_t t = threadIdx.x; t <= a.rows; t += 256)
      if (t != r)
        a.out_tokens[trow + t] = t < r ? a.tokens[(size_t)b * a.rows + t] : 0xFFFFFFFFu;
    if (threadIdx.x == 0) a.out_counts[b] = r + 1;
  }
  if (greedy) {
    if (part == 0 && threadIdx.x == 0) a.out_tokens[trow + r] = dec.first;
    return;
  }
  double sr = 0.0, sf = 0.0;
  for (int i = 0; i < kPer; ++i) {
    const uint32_t id = part * kPart + i * 256 + threadIdx.x;
    if (id >= a.n) break;
    double x, y;
    id_weights(a, dec, b, id, inv_t, x, y);
    sr += x;
    sf += y;
  }
  sr = block_sum_f64(sr, red);
  sf = block_sum_f64(sf, red);
  if (threadIdx.x == 0) rest[blockIdx.x] = make_double2(sr, sf);
}

__global__ __launch_bounds__(256) void k_verify_pick(VerifyArgs a, const double2* rest,
                                                     const Decision* decisions, int parts) {
  const uint32_t b = blockIdx.x;
  const Decision d = decisions[b];
  const double inv_t = 1.0 / (double)a.temperature;
  const double2* s = rest + (size_t)b * parts;
  __shared__ double before[256];
  __shared__ uint32_t found, last;
  // Every thread walks the parts' few sums alike.
  double sr = 0.0, sf = 0.0;
  for (int i = 0; i < parts; ++i) {
    sr += s[i].x;
    sf += s[i].y;
  }
  const bool use_rest = sr > 0.0;
  const double total = use_rest ? sr : sf;
  if (!(total > 0.0)) {
    if (threadIdx.x == 0) a.out_tokens[(size_t)b * (a.rows + 1) + d.row] = d.first;
    return;
  }
  const double point = a.uniforms[(size_t)b * (a.rows + 1) + a.rows] * total;
  double sum = 0.0, base = 0.0;
  int part = 0;
  for (int i = 0; i < parts; ++i) {
    const double w = use_rest ? s[i].x : s[i].y;
    if (w > 0.0 && sum <= point) {  // the last part that begins at or before the point
      part = i;
      base = sum;
    }
    sum += w;
  }
  // Sixteen consecutive ids per thread.
  const uint32_t id0 = part * kPart + threadIdx.x * kPer;
  double w[kPer], own = 0.0;
  for (int i = 0; i < kPer; ++i) {
    w[i] = 0.0;
    if (id0 + i < a.n) {
      double x, y;
      id_weights(a, d, b, id0 + i, inv_t, x, y);
      w[i] = use_rest ? x : y;
    }
    own += w[i];
  }
  before[threadIdx.x] = own;
  if (threadIdx.x == 0) {
    found = 0xFFFFFFFFu;
    last = 0;
  }
  __syncthreads();
  double cum = base;
  for (int i = 0; i < (int)threadIdx.x; ++i) cum += before[i];
  // The first id whose cumulative weight exceeds the point; where rounding
  // leaves none, the last one with weight.
  uint32_t mine = 0xFFFFFFFFu, weighty = 0xFFFFFFFFu;
  for (int i = 0; i < kPer; ++i) {
    cum += w[i];
    if (w[i] > 0.0) {
      weighty = id0 + i;
      if (cum > point && mine == 0xFFFFFFFFu) mine = id0 + i;
    }
  }
  if (mine != 0xFFFFFFFFu) atomicMin(&found, mine);
  if (weighty != 0xFFFFFFFFu) atomicMax(&last, weighty);
  __syncthreads();
  if (threadIdx.x == 0)
    a.out_tokens[(size_t)b * (a.rows + 1) + d.row] = found != 0xFFFFFFFFu ? found : last;
}

int parts_of(uint32_t n) { return (int)((n + kPart - 1) / kPart); }
uint64_t stat_rows(uint32_t batch, uint32_t rows) { return (uint64_t)batch * (2 * (uint64_t)rows + 1); }

}  // namespace

uint64_t verify_blocks(uint32_t batch, uint32_t rows, uint32_t n) {
  return stat_rows(batch, rows) * parts_of(n);
}

size_t verify_workspace_bytes(uint32_t batch, uint32_t rows, uint32_t n) {
  return verify_blocks(batch, rows, n) * sizeof(PartStat) +
         (size_t)batch * parts_of(n) * sizeof(double2) + (size_t)batch * sizeof(Decision);
}

hipError_t launch_verify(const VerifyArgs& a, hipStream_t s) {
  const int parts = parts_of(a.n);
  PartStat* stats = static_cast<PartStat*>(a.ws);
  double2* rest = reinterpret_cast<double2*>(stats + verify_blocks(a.batch, a.rows, a.n));
  Decision* dec = reinterpret_cast<Decision*>(rest + (size_t)a.batch * parts);
  const uint64_t rows = a.draft ? stat_rows(a.batch, a.rows) : (uint64_t)a.batch * (a.rows + 1);
  hipLaunchKernelGGL(k_verify_stats, dim3((uint32_t)(rows * parts)), dim3(256), 0, s, a, stats,
                     parts);
  hipLaunchKernelGGL(k_verify_rest, dim3((uint32_t)(a.temperature > 0.f ? a.batch * parts : a.batch)),
                     dim3(256), 0, s, a, stats, rest, dec, parts);
  if (a.temperature > 0.f)
    hipLaunchKernelGGL(k_verify_pick, dim3(a.batch), dim3(256), 0, s, a, rest, dec, parts);
  return hipGetLastError();
}

}  // namespace akh
