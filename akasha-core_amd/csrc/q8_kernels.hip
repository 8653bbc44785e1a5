// 8-bit KV caches: rows quantised as they are written, read back, and
// attended to (akh_cache_write_q8, akh_cache_read_q8, akh_attn_*_q8).
//
// A head's row is int8 codes and one power of two: the scaling is exact both
// ways, so a value has seen a single rounding, and every kernel here works on
// the same values whatever order it reads them in.
#include <hip/hip_runtime.h>

#include "common.h"
#include "kernels.h"

namespace akh {

namespace {

constexpr int kNanExp = -128;  // exponent of a row with a NaN or an infinity

// 2^e of a cache exponent, NaN for kNanExp.
__device__ __forceinline__ float exp_value(int e) {
  return e == kNanExp ? __int_as_float(0x7FC00000) : __int_as_float((e + 127) << 23);
}

// Rows of this step in sequence b.
__device__ __forceinline__ uint32_t step_rows(const uint32_t* counts, uint32_t b, uint32_t rows) {
  return counts ? min(counts[b], rows) : rows;
}

// Maximum over aligned groups of N lanes (16 or 32), every lane active.
template <int N>
__device__ __forceinline__ uint32_t group_umax(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, true));
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xF, 0xF, true));
  if constexpr (N == 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max((uint32_t)r[0], (uint32_t)r[1]);
  }
  return v;
}

// One item is one head's row of K or V: ROW / 4 lanes of four columns each.
// Items run over heads first, so a wave reads consecutive columns.
struct Q8Item {
  uint32_t b, t, head;
  bool is_v;
};
__device__ __forceinline__ Q8Item q8_item(uint64_t id, uint32_t rows, uint32_t kv_heads) {
  Q8Item it;
  it.head = (uint32_t)(id % kv_heads);
  id /= kv_heads;
  it.is_v = id & 1;
  id >>= 1;
  it.t = (uint32_t)(id % rows);
  it.b = (uint32_t)(id / rows);
  return it;
}

template <int ROW, bool VEC>
__global__ __launch_bounds__(256) void k_cache_write_q8(const float* k, const float* v,
                                                        Q8Cache c, uint32_t batch, uint32_t rows,
                                                        uint32_t stride, const uint32_t* pos,
                                                        const uint32_t* counts) {
  constexpr int L = ROW / 4;
  const int col = (threadIdx.x % L) * 4;
  const uint64_t items = (uint64_t)batch * rows * 2 * c.kv_heads;
  const uint64_t id = (uint64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  if (id >= items) return;  // whole groups of L lanes leave together
  const Q8Item it = q8_item(id, rows, c.kv_heads);
  const uint64_t at = (uint64_t)pos[it.b] + it.t;
  if (it.t >= step_rows(counts, it.b, rows) || at >= c.max_rows) return;
  const float* src = (it.is_v ? v : k) + ((size_t)it.b * rows + it.t) * stride +
                     (size_t)it.head * c.head_dim;
  float x[4];
  if constexpr (VEC) {
    const float4 f = col < (int)c.head_dim ? *reinterpret_cast<const float4*>(src + col)
                                           : make_float4(0.f, 0.f, 0.f, 0.f);
    x[0] = f.x;
    x[1] = f.y;
    x[2] = f.z;
    x[3] = f.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = col + i < (int)c.head_dim ? src[col + i] : 0.f;
  }
  uint32_t top = 0;  // magnitudes order as their bits, infinities and NaN above all
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  top = group_umax<L>(top);
  // top = 1.m * 2^(E - 127); 127 * 2^e = (127 / 64) * 2^(e + 6), and 1.m <=
  // 127 / 64 is m <= 0x7E0000.
  const bool bad = top >= 0x7F800000u;
  const int e = max(-126, (int)(top >> 23) - 133 + ((top & 0x7FFFFFu) > 0x7E0000u));
  const float inv = __int_as_float((127 - e) << 23);
  const float most = e == 122 ? 63.f : 127.f;  // 64 * 2^122 would read back as infinity
  uint32_t packed = 0;
  if (!bad) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      packed |= (uint32_t)((int)fminf(fmaxf(rintf(x[i] * inv), -most), most) & 0xFF) << (8 * i);
  }
  const size_t row = ((size_t)it.b * c.kv_heads + it.head) * c.cap + at;
  *reinterpret_cast<uint32_t*>((it.is_v ? c.v : c.k) + row * ROW + col) = packed;
  if (col == 0) (it.is_v ? c.ve : c.ke)[row] = (int8_t)(bad ? kNanExp : e);
}

template <int ROW, bool VEC>
__global__ __launch_bounds__(256) void k_cache_read_q8(Q8Cache c, float* k, float* v,
                                                       uint32_t batch, uint32_t rows,
                                                       uint32_t stride, const uint32_t* pos,
                                                       const uint32_t* counts) {
  constexpr int L = ROW / 4;
  const int col = (threadIdx.x % L) * 4;
  const uint64_t items = (uint64_t)batch * rows * 2 * c.kv_heads;
  const uint64_t id = (uint64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  if (id >= items || col >= (int)c.head_dim) return;
  const Q8Item it = q8_item(id, rows, c.kv_heads);
  float* dst = it.is_v ? v : k;
  if (!dst) return;
  dst += ((size_t)it.b * rows + it.t) * stride + (size_t)it.head * c.head_dim + col;
  const uint64_t at = (uint64_t)pos[it.b] + it.t;
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  if (it.t < step_rows(counts, it.b, rows) && at < c.max_rows) {
    const size_t row = ((size_t)it.b * c.kv_heads + it.head) * c.cap + at;
    const uint32_t q =
        *reinterpret_cast<const uint32_t*>((it.is_v ? c.v : c.k) + row * ROW + col);
    const float s = exp_value((it.is_v ? c.ve : c.ke)[row]);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(q >> (8 * i)) * s;
  }
  if constexpr (VEC) {
    *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (col + i < (int)c.head_dim) dst[i] = x[i];
  }
}

// One block per (sequence, row, head): four waves deal the keys of the
// prefix and of the sequence's own rows among them, a lane holds ROW / 64
// columns, and the waves' running maxima, sums and weighted rows are joined
// at the end.
template <int ROW>
__global__ __launch_bounds__(256) void k_attn_q8(AttnQ8Args a) {
  constexpr int D = ROW / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t h = blockIdx.x % a.heads;
  const uint64_t bt = blockIdx.x / a.heads;
  const uint32_t b = (uint32_t)(bt / a.rows), t = (uint32_t)(bt % a.rows);
  const uint32_t kvh = h / (a.heads / a.c.kv_heads);
  float* out = a.out + bt * a.out_stride + (size_t)h * a.c.head_dim;
  const bool live = t < step_rows(a.counts, b, a.rows);
  const uint32_t own =
      live ? (uint32_t)min<uint64_t>((uint64_t)a.pos[b] + t + 1, a.c.max_rows) : 0;
  const uint32_t ahead = live && a.prefix_len ? min(*a.prefix_len, a.pre.max_rows) : 0;
  float q[D], acc[D];
#pragma unroll
  for (int i = 0; i < D; ++i) {
    const int col = lane * D + i;
    q[i] = col < (int)a.c.head_dim ? a.q[bt * a.q_stride + (size_t)h * a.c.head_dim + col] : 0.f;
    acc[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (uint64_t j = wave; j < (uint64_t)ahead + own; j += 4) {
    const bool first = j < ahead;
    const Q8Cache& c = first ? a.pre : a.c;
    const size_t row = ((size_t)(first ? 0 : b) * c.kv_heads + kvh) * c.cap + (first ? j : j - ahead);
    float s = 0.f, vv[D];
#pragma unroll
    for (int i = 0; i < D; ++i) {
      s = fmaf(q[i], (float)c.k[row * ROW + lane * D + i], s);
      vv[i] = (float)c.v[row * ROW + lane * D + i];
    }
    s = wave_sum(s) * exp_value(c.ke[row]) * a.scale;
    const float mn = fmaxf(m, s);
    const float keep = m == -INFINITY ? 0.f : expf(m - mn);
    const float p = mn == -INFINITY && s == -INFINITY ? 0.f : expf(s - mn);
    const float w = p * exp_value(c.ve[row]);
    l = l * keep + p;
#pragma unroll
    for (int i = 0; i < D; ++i) acc[i] = acc[i] * keep + w * vv[i];
    m = mn;
  }
  __shared__ float sm[4], sl[4], sa[4][ROW];
  if (lane == 0) {
    sm[wave] = m;
    sl[wave] = l;
  }
#pragma unroll
  for (int i = 0; i < D; ++i) sa[wave][lane * D + i] = acc[i];
  __syncthreads();
  const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float f[4], total = 0.f;
  for (int w = 0; w < 4; ++w) {
    f[w] = sm[w] == -INFINITY ? (sl[w] == sl[w] ? 0.f : 1.f) : expf(sm[w] - top);
    total += sl[w] * f[w];
  }
  if (threadIdx.x < a.c.head_dim) {
    float x = 0.f;
    for (int w = 0; w < 4; ++w) x += sa[w][threadIdx.x] * f[w];
    out[threadIdx.x] = own || ahead ? x / total : 0.f;
  }
  if (threadIdx.x == 0 && a.lse)
    a.lse[bt * a.heads + h] = own || ahead ? top + logf(total) : -INFINITY;
}

uint64_t div_up(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

bool vec4(const void* p, uint32_t stride, uint32_t head_dim) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % 4 == 0 && head_dim % 4 == 0;
}

}  // namespace

hipError_t launch_cache_write_q8(const float* k, const float* v, const Q8Cache& c, uint32_t batch,
                                 uint32_t rows, uint32_t stride, const uint32_t* pos,
                                 const uint32_t* counts, hipStream_t s) {
  const bool vec = vec4(k, stride, c.head_dim) && vec4(v, stride, c.head_dim);
  const bool wide = c.row == 128;
  const uint64_t items = (uint64_t)batch * rows * 2 * c.kv_heads;
  const dim3 grid((uint32_t)div_up(items, wide ? 8 : 16));
  auto* f = wide ? (vec ? k_cache_write_q8<128, true> : k_cache_write_q8<128, false>)
                 : (vec ? k_cache_write_q8<64, true> : k_cache_write_q8<64, false>);
  hipLaunchKernelGGL(f, grid, dim3(256), 0, s, k, v, c, batch, rows, stride, pos, counts);
  return hipGetLastError();
}

hipError_t launch_cache_read_q8(const Q8Cache& c, float* k, float* v, uint32_t batch,
                                uint32_t rows, uint32_t stride, const uint32_t* pos,
                                const uint32_t* counts, hipStream_t s) {
  const bool vec = (!k || vec4(k, stride, c.head_dim)) && (!v || vec4(v, stride, c.head_dim));
  const bool wide = c.row == 128;
  const uint64_t items = (uint64_t)batch * rows * 2 * c.kv_heads;
  const dim3 grid((uint32_t)div_up(items, wide ? 8 : 16));
  auto* f = wide ? (vec ? k_cache_read_q8<128, true> : k_cache_read_q8<128, false>)
                 : (vec ? k_cache_read_q8<64, true> : k_cache_read_q8<64, false>);
  hipLaunchKernelGGL(f, grid, dim3(256), 0, s, c, k, v, batch, rows, stride, pos, counts);
  return hipGetLastError();
}

size_t attn_q8_workspace_bytes(const AttnQ8Args&) { return 0; }

hipError_t launch_attn_q8(const AttnQ8Args& a, hipStream_t s) {
  const dim3 grid((uint32_t)((uint64_t)a.batch * a.rows * a.heads));
  hipLaunchKernelGGL(a.c.row == 128 ? k_attn_q8<128> : k_attn_q8<64>, grid, dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace akh
