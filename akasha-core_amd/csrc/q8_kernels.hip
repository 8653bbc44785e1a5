// 8-bit KV caches: rows quantised as they are written, read back, and
// attended to (akh_cache_write_q8, akh_cache_read_q8, akh_attn_*_q8).
//
// A head's row is int8 codes and one power of two: the scaling is exact both
// ways, so a value has seen a single rounding, and every kernel here works on
// the same values whatever order it reads them in.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

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

// Rows in and out of the cache.  A head's row of K or V is a group of ROW / 4
// lanes of four columns each; a block takes 1024 / ROW consecutive heads (K's, then V's) of
// R consecutive rows of one sequence, so a thread has R loads under way and a
// wave's are whole lines.  Bound by memory: of 8 x 2040 rows of 16 heads of 128
// with 10987 rows live (180 MB of f32 and 45 of codes; the read fills all 267 MB)
// the write takes 43 us and the read 45.  Both together were 145 us with a row a
// thread, 114 with four, and are 88 with f32 past the caches.
struct Q8Rows {
  uint32_t batch, rows, stride, groups, blocks;  // groups of R rows, blocks of a row's heads
  const uint32_t* pos;
  const uint32_t* counts;
};
struct Q8Place {
  uint32_t b, t0, head, live;  // live: rows of the step
  uint64_t at;                 // of row t0 in the cache
  bool is_v, in;
};
template <int ROW, int R>
__device__ __forceinline__ Q8Place q8_place(const Q8Rows& a, const Q8Cache& c) {
  Q8Place p;
  uint32_t id = blockIdx.x;
  uint32_t block = 0;
  if (a.blocks > 1) {
    block = id % a.blocks;
    id /= a.blocks;
  }
  uint32_t group = 0;
  if (a.groups > 1) {
    group = id % a.groups;
    id /= a.groups;
  }
  p.b = id;
  p.t0 = group * R;
  const uint32_t item = block * (1024 / ROW) + threadIdx.x / (ROW / 4);
  p.is_v = item >= c.kv_heads;
  p.head = p.is_v ? item - c.kv_heads : item;
  p.in = p.head < c.kv_heads;
  p.live = step_rows(a.counts, p.b, a.rows);
  p.at = (uint64_t)a.pos[p.b] + p.t0;
  return p;
}

template <int ROW, int R, bool VEC>
__global__ __launch_bounds__(256) void k_cache_write_q8(const float* k, const float* v,
                                                        Q8Cache c, Q8Rows a) {
  const int col = threadIdx.x % (ROW / 4) * 4;
  const Q8Place p = q8_place<ROW, R>(a, c);
  if (!p.in || p.t0 >= p.live || p.at >= c.max_rows) return;  // a group's lanes alike
  const uint32_t n = (uint32_t)min<uint64_t>(min(R, (int)(p.live - p.t0)), c.max_rows - p.at);
  const float* src = (p.is_v ? v : k) + ((size_t)p.b * a.rows + p.t0) * a.stride +
                     (size_t)p.head * c.head_dim;
  float x[R][4];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const float* row = src + (size_t)min((uint32_t)i, n - 1) * a.stride;
    if constexpr (VEC) {
      typedef float f4 __attribute__((ext_vector_type(4)));
      const f4 f = __builtin_nontemporal_load(reinterpret_cast<const f4*>(row + min(col, (int)c.head_dim - 4)));
      x[i][0] = f.x;
      x[i][1] = f.y;
      x[i][2] = f.z;
      x[i][3] = f.w;
    } else {
#pragma unroll
      for (int d = 0; d < 4; ++d) x[i][d] = row[min(col + d, (int)c.head_dim - 1)];
    }
  }
  const size_t row0 = ((size_t)p.b * c.kv_heads + p.head) * c.cap + p.at;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    uint32_t top = 0;  // magnitudes order as their bits, infinities and NaN above all
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      if (col + d >= (int)c.head_dim) x[i][d] = 0.f;
      top = max(top, __float_as_uint(x[i][d]) & 0x7FFFFFFFu);
    }
    top = group_umax<ROW / 4>(top);
    // top = 1.m * 2^(E - 127); 127 * 2^e = (127 / 64) * 2^(e + 6), and 1.m <=
    // 127 / 64 is m <= 0x7E0000.
    const bool bad = top >= 0x7F800000u;
    const int e = max(-126, (int)(top >> 23) - 133 + ((top & 0x7FFFFFu) > 0x7E0000u));
    const float inv = __int_as_float((127 - e) << 23);
    const float most = e == 122 ? 63.f : 127.f;  // 64 * 2^122 would read back as infinity
    uint32_t packed = 0;
    if (!bad) {
#pragma unroll
      for (int d = 0; d < 4; ++d)
        packed |= (uint32_t)((int)fminf(fmaxf(rintf(x[i][d] * inv), -most), most) & 0xFF)
                  << (8 * d);
    }
    if (i < (int)n) {
      *reinterpret_cast<uint32_t*>((p.is_v ? c.v : c.k) + (row0 + i) * ROW + col) = packed;
      if (col == 0) (p.is_v ? c.ve : c.ke)[row0 + i] = (int8_t)(bad ? kNanExp : e);
    }
  }
}

template <int ROW, int R, bool VEC>
__global__ __launch_bounds__(256) void k_cache_read_q8(Q8Cache c, float* k, float* v, Q8Rows a) {
  const int col = threadIdx.x % (ROW / 4) * 4;
  const Q8Place p = q8_place<ROW, R>(a, c);
  float* dst = p.is_v ? v : k;
  if (!p.in || !dst || col >= (int)c.head_dim) return;
  dst += ((size_t)p.b * a.rows + p.t0) * a.stride + (size_t)p.head * c.head_dim + col;
  // Rows held, of R; the others become zero.
  const uint32_t n = p.t0 < p.live && p.at < c.max_rows
                         ? (uint32_t)min<uint64_t>(min(R, (int)(p.live - p.t0)), c.max_rows - p.at)
                         : 0;
  const size_t row0 = ((size_t)p.b * c.kv_heads + p.head) * c.cap + (n ? p.at : 0);
  uint32_t q[R];
  int e[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const size_t row = row0 + min((uint32_t)i, n ? n - 1 : 0);
    q[i] = *reinterpret_cast<const uint32_t*>((p.is_v ? c.v : c.k) + row * ROW + col);
    e[i] = (p.is_v ? c.ve : c.ke)[row];
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (p.t0 + i >= a.rows) break;
    const float s = exp_value(e[i]);
    float x[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) x[d] = i < (int)n ? (float)(int8_t)(q[i] >> (8 * d)) * s : 0.f;
    float* out = dst + (size_t)i * a.stride;
    if constexpr (VEC) {
      typedef float f4 __attribute__((ext_vector_type(4)));
      __builtin_nontemporal_store(f4{x[0], x[1], x[2], x[3]}, reinterpret_cast<f4*>(out));
    } else {
#pragma unroll
      for (int d = 0; d < 4; ++d)
        if (col + d < (int)c.head_dim) out[d] = x[d];
    }
  }
}

// ---- attention ---------------------------------------------------------------
//
// A job is one kv head's keys of one source (a sequence's slot, or the
// prefix), a group of the query rows that read them, and one of the splits of
// those keys.  Its block's waves deal the split's 32-key tiles among them and
// go through each tile once, with the softmax's running maximum and sum:
//
//   S^T = K Q^T      16x16x32 fp16 MFMAs, A = K's codes, B = the rows' q
//   P^T = 2^(S - m)  in the accumulators' layout, which is already B's
//   O^T += V^T P^T   A = V's codes by dimension
//
// int8 codes are exact in fp16, q and P go in as two fp16 terms each, hi + lo
// (22 bits).  With at most 8 rows the terms are two columns of one MFMA (PACK:
// column c is row c's hi, c + 8 its lo); otherwise two MFMAs into one
// accumulator, 16 rows a tile, NT tiles.
//
// Lane l = 16 g + c.  K: the lane holds 16 columns of key c (16 g + 64 u
// ..), which two MFMA steps contract in that order, q's alike.  S^T: rows
// (keys) 4 g + r of both 16-key halves, column c.  P^T as B wants keys 8 g
// + i of a 32-key contraction: keys are taken in the order 4 g + r, 16 + 4 g + r,
// so P never leaves its lane; V's codes come in the same order, the lane's
// ROW / 16 consecutive columns of eight keys: column (ROW / 16) c + j is A's
// row c of MFMA j.
//
// The exponents: a key's K scale multiplies its scores, its V scale its
// weights.  Sums add 2^(x - mt), products take w = 2^(x - mt) 2^(ve - ev), with
// whole mt and ev of each row, from the keys that it sees, such that its largest w
// lies at 2^-4; w may grow to 2^15 (PACK: 61440) before they move and the
// accumulators are rescaled (exactly), so most tiles neither join maxima across
// lanes nor rescale.  Mostly ev is 0: one 2^x serves both.  Where mt would then lie
// 2^90 below the row's largest score, or a V scale of 2^90 meets 2^x below 32 bits'
// normal range, the wave's rows are kept apart: mt by the scores alone, and w by a
// 2^x of its own.  lo is kept times 2^11 and meets V's codes times 2^-11 (PACK: its
// column's results take the factor), so a weight loses what is below 2^-36 (PACK,
// which truncates lo: 2^-35) only, next to a largest one above 2^-5.  With lo
// unscaled and levels at 2^6 the 32 rows of a
// wave moved them so often that the barriers of blocks in LDS waited for one
// wave or another: 69 us in place of 64 behind 8200 keys whose scales differ by 16.

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Bytes 0, 1 and 2, 3 of four offset codes (code + 128) as fp16 codes: under
// the exponent byte 0x64 a byte reads 1024 + it.
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const h2 off = {(_Float16)-1152.f, (_Float16)-1152.f};
  w ^= 0x80808080u;
  lo = __builtin_bit_cast(
      uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + off);
  hi = __builtin_bit_cast(
      uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + off);
}
__device__ __forceinline__ f16x8 codes8_f16(uint32_t a, uint32_t b) {
  uint4 r;
  codes_f16(a, r.x, r.y);
  codes_f16(b, r.z, r.w);
  return f16x8_of(r);
}
// Byte J of two dwords as a pair of fp16 codes.
template <int J>
__device__ __forceinline__ uint32_t pair_f16(uint32_t a, uint32_t b) {
  const h2 off = {(_Float16)-1152.f, (_Float16)-1152.f};
  const uint32_t w = __builtin_amdgcn_perm(b, a, 0x0C040C00u + J * 0x00010001u) ^ 0x64806480u;
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, w) + off);
}

// Two floats of at most 2^15 as hi + lo fp16 pairs: hi truncated to 11
// bits, lo the rest rounded to 11 (together within 2^-22, or 2^-25 below fp16's
// normal range).
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  const h2 h = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(a, b));
  const h2 l = {(_Float16)fmaf((float)h[0], -1.f, a), (_Float16)fmaf((float)h[1], -1.f, b)};
  hi = __builtin_bit_cast(uint32_t, h);
  lo = __builtin_bit_cast(uint32_t, l);
}
// The same with lo times 2^11 (a, b at most 2^15), for weights: it keeps what lies below hi of
// the smallest ones too.
__device__ __forceinline__ void split2_up(float a, float b, uint32_t& hi, uint32_t& lo) {
  const h2 h = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(a, b));
  const h2 l = {(_Float16)fmaf((float)h[0], -2048.f, a * 2048.f),
                (_Float16)fmaf((float)h[1], -2048.f, b * 2048.f)};
  hi = __builtin_bit_cast(uint32_t, h);
  lo = __builtin_bit_cast(uint32_t, l);
}

__device__ __forceinline__ int byte_s(uint32_t w, int i) { return (int)(int8_t)(w >> (8 * i)); }
typedef int i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ i32x4 exps_of(uint32_t w) {
  return i32x4{byte_s(w, 0), byte_s(w, 1), byte_s(w, 2), byte_s(w, 3)};
}
// K exponents from here on are applied next to q's (2^29 codes times more may leave f32), V's
// of rows kept apart.
constexpr int kBigExp = 90;
// In the place of q's exponent for rows that are not there: they weigh every key alike, so that
// their scores move no levels.
constexpr int kNoRow = -1000;
__device__ __forceinline__ bool outside_f32(int qx) {
  return qx != kNoRow && (qx < -126 || qx > 127);
}

// What one 32-key tile's lane loads.
template <int ROW>
struct Tile {
  uint4 k[2][ROW / 64];
  uint32_t v[8][ROW / 64];
  uint32_t ke[2], ve[2];
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
// STREAM: past the caches, for codes that will not be met there again.
template <bool STREAM, class T>
__device__ __forceinline__ T load_codes(const int8_t* p) {
  if constexpr (STREAM)
    return __builtin_nontemporal_load(reinterpret_cast<const T*>(p));
  else
    return *reinterpret_cast<const T*>(p);
}
template <int ROW, bool STREAM>
__device__ __forceinline__ void load_k(Tile<ROW>& t, const int8_t* k, const int8_t* ke,
                                       const int8_t* ve, uint32_t key0, int g, int c) {
  const int8_t* kp = k + (size_t)(key0 + c) * ROW + 16 * g;
#pragma unroll
  for (int hh = 0; hh < 2; ++hh) {
#pragma unroll
    for (int u = 0; u < ROW / 64; ++u)
      t.k[hh][u] = __builtin_bit_cast(
          uint4, load_codes<STREAM, u32x4>(kp + hh * 16 * ROW + u * 64));
    t.ke[hh] = *reinterpret_cast<const uint32_t*>(ke + key0 + 16 * hh + 4 * g);
    t.ve[hh] = *reinterpret_cast<const uint32_t*>(ve + key0 + 16 * hh + 4 * g);
  }
}
template <int ROW, bool STREAM>
__device__ __forceinline__ void load_v(Tile<ROW>& t, const int8_t* v, uint32_t key0, int g,
                                       int c) {
  const int8_t* vp = v + (size_t)(key0 + 4 * g) * ROW + c * (ROW / 16);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int8_t* p = vp + ((i & 3) + (i >> 2) * 16) * ROW;
    if constexpr (ROW == 64) {
      t.v[i][0] = load_codes<STREAM, uint32_t>(p);
    } else {
      const u32x2 w = load_codes<STREAM, u32x2>(p);
      t.v[i][0] = w.x;
      t.v[i][1] = w.y;
    }
  }
}

// One query row of a job.
struct RowRef {
  uint64_t bt;     // row of q and out
  uint32_t head;
  uint32_t limit;  // keys it sees
  bool live;       // it is the step's (otherwise it sees no key)
};

// A job's place, and what its rows see.
template <bool SHARED>
struct Job {
  uint32_t b, kvh, group, split, splits, nrows, G;
  uint32_t live_rows;  // of the sequence; SHARED: unused
  uint32_t pos;
  uint32_t keys;       // the prefix's

  __device__ __forceinline__ void init(const AttnQ8Args& a, const AttnQ8Plan& pl) {
    uint32_t id = blockIdx.x;
    const uint32_t groups = SHARED ? pl.prefix_groups : pl.own_groups;
    splits = SHARED ? pl.prefix_splits : pl.own_splits;
    G = pl.G;
    group = 0;
    if (groups > 1) {
      // Blocks go to the eight XCDs in turn: those of the same keys to one, for its L2.
      const uint32_t even = gridDim.x / groups / 8 * 8;
      if (id < even * groups) {
        const uint32_t k = id / 8;
        group = k % groups;
        id = k / groups * 8 + id % 8;
      } else {
        id -= even * groups;
        group = id % groups;
        id = even + id / groups;
      }
    }
    kvh = id % a.c.kv_heads;
    id /= a.c.kv_heads;
    split = 0;
    if (SHARED) {
      split = id;
    } else if (splits > 1) {
      split = id % splits;
      id /= splits;
    }
    b = SHARED ? 0 : id;
    nrows = (SHARED ? a.batch : 1) * a.rows * G;
    if constexpr (SHARED) {
      keys = min(*a.prefix_len, a.pre.max_rows);
    } else {
      live_rows = step_rows(a.counts, b, a.rows);
      pos = a.pos[b];
    }
  }
  __device__ __forceinline__ uint32_t sees(const AttnQ8Args& a, uint32_t t) const {
    return (uint32_t)min<uint64_t>((uint64_t)pos + t + 1, a.c.max_rows);
  }
  // Row r of the job's kv head, G query heads each (SHARED: of every sequence).
  __device__ __forceinline__ RowRef row(const AttnQ8Args& a, uint32_t r) const {
    RowRef x;
    x.live = r < nrows;
    r = min(r, nrows - 1);
    uint32_t t = r, h = 0, s = b;
    if (G > 1) {
      t = r / G;
      h = r - t * G;
    }
    if constexpr (SHARED) {
      s = t;
      if (a.rows > 1) s = t / a.rows;
      t -= s * a.rows;
      x.live = x.live && t < step_rows(a.counts, s, a.rows);
      x.limit = x.live ? keys : 0;
    } else {
      x.live = x.live && t < live_rows;
      x.limit = x.live ? sees(a, t) : 0;
    }
    x.head = kvh * G + h;
    x.bt = (uint64_t)s * a.rows + t;
    return x;
  }
  // Keys that any (most) and every live row (least) of rows row0 .. + n - 1
  // sees.
  __device__ __forceinline__ void span(const AttnQ8Args& a, uint32_t row0, uint32_t n,
                                       uint32_t& least, uint32_t& most) const {
    if constexpr (SHARED) {
      least = most = keys;
    } else {
      uint32_t first = row0, last = min(row0 + n, nrows) - 1;
      if (G > 1) {
        first /= G;
        last /= G;
      }
      const bool some = row0 < nrows && first < live_rows;
      least = some ? sees(a, first) : 0xFFFFFFFFu;
      most = some ? sees(a, min(last, live_rows - 1)) : 0;
    }
  }
};

// q of one row, as the lane's columns of the MFMA steps.
template <int ROW>
struct RawQ {
  float x[ROW / 32][8];

  __device__ __forceinline__ void load(const AttnQ8Args& a, const RowRef& r, int g) {
    const float* q = a.q + r.bt * a.q_stride + (size_t)r.head * a.c.head_dim;
    const int hd = (int)a.c.head_dim;
    if (a.q_vec) {  // head_dim is a multiple of 4
#pragma unroll
      for (int s = 0; s < ROW / 32; ++s)
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          const int d = (s >> 1) * 64 + 16 * g + 8 * (s & 1) + i;
          const float4 u = *reinterpret_cast<const float4*>(q + min(d, hd - 4));
          x[s][i] = u.x;
          x[s][i + 1] = u.y;
          x[s][i + 2] = u.z;
          x[s][i + 3] = u.w;
        }
    } else {
#pragma unroll
      for (int s = 0; s < ROW / 32; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          x[s][i] = q[min((s >> 1) * 64 + 16 * g + 8 * (s & 1) + i, hd - 1)];
    }
    if (hd != ROW) {
#pragma unroll
      for (int s = 0; s < ROW / 32; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if ((s >> 1) * 64 + 16 * g + 8 * (s & 1) + i >= hd) x[s][i] = 0.f;
    }
  }

  // The same from 16 rows in LDS, `rs` floats apart.
  __device__ __forceinline__ void from_lds(const float* rows, int rs, int g, int c) {
#pragma unroll
    for (int s = 0; s < ROW / 32; ++s)
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const f32x4 u = *reinterpret_cast<const f32x4*>(
            rows + c * rs + (s >> 1) * 64 + 16 * g + 8 * (s & 1) + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[s][i + k] = u[k];
      }
  }

  // As B operands, hi and lo, times scale log2(e) 2^-e with a largest magnitude
  // in [2^13, 2^14]; returns e.  The scale comes as mantissa and exponent, so that
  // its product with q does not leave f32.  A NaN or an infinity makes one
  // of the terms NaN (inf - inf), and with it the row's scores.
  __device__ __forceinline__ int operands(const AttnQ8Args& a, f16x8* hi, f16x8* lo) {
    float top = 0.f;
#pragma unroll
    for (int s = 0; s < ROW / 32; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[s][i]));
    top = xor_max<32>(xor_max<16>(top));
    const float m = __builtin_amdgcn_frexp_mantf(top) * fabsf(a.scale_mant);
    const int up = 14 - __builtin_amdgcn_frexp_expf(top) + (m < 0.5f);
    const int first = up > 126 ? up - 126 : 0;  // of the smallest rows, whose factor leaves f32
    if (__builtin_expect(__any(first != 0), 0)) {
      asm volatile("");
#pragma unroll
      for (int s = 0; s < ROW / 32; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[s][i] = ldexpf(x[s][i], first);
    }
    const float f = ldexpf(a.scale_mant, up - first);
#pragma unroll
    for (int s = 0; s < ROW / 32; ++s) {
      uint32_t h[4], l[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) split2(x[s][2 * i] * f, x[s][2 * i + 1] * f, h[i], l[i]);
      hi[s] = f16x8_of(make_uint4(h[0], h[1], h[2], h[3]));
      lo[s] = f16x8_of(make_uint4(l[0], l[1], l[2], l[3]));
    }
    return a.scale_exp - up;
  }
};

// Partial results of a row: maximum (log2), sum and normalised weighted row
// of each part; the prefix's splits first, then the own rows'.
struct PartMl {
  float m, l;
};
// A part's sum next to level `top`.  Levels are whole numbers, and those of parts whose V scales
// are far apart may differ by 2^184 where their sums do by the inverse: as a factor, 2^(m - top)
// could leave f32.
__device__ __forceinline__ float part_sum(const PartMl& p, float top) {
  return p.l == 0.f ? 0.f : ldexpf(p.l, (int)fmaxf(p.m - top, -1000.f));
}
__device__ __forceinline__ size_t row_id(const AttnQ8Args& a, const RowRef& r) {
  return r.bt * a.heads + r.head;
}

// A wave's rows on their way over the keys.
template <int ROW, int NT>
struct RowsState {
  f32x4 acc[NT][ROW / 16];
  float mt[NT], ev[NT], l[NT];
  bool fresh, apart;  // of the wave; ev is 0 unless apart

  __device__ __forceinline__ void init() {
    fresh = true;
    apart = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      mt[n] = ev[n] = 0.f;
      l[n] = 0.f;
#pragma unroll
      for (int j = 0; j < ROW / 16; ++j) acc[n][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
};

// One tile of 32 keys: kfrag(hh, s) and vfrag(j) give K's and V's A operands,
// kexp(hh) and vexp(hh) the exponents of the lane's four keys of half hh (any number
// in range behind the last key that any row sees), odd whether the tile has a NaN
// row or an exponent of kBigExp, or a row a q exponent outside f32.  qx(n): exponents of q's
// operands, kNoRow for rows that are not there.  limit: keys a row sees; a tile past the least
// of them needs the mask.  k_used() is called once K's operands are spent.
template <int ROW, int NT, bool PACK, class QX, class KF, class VF, class KE, class VE,
          class HK>
__device__ __forceinline__ void tile_step(RowsState<ROW, NT>& st, const f16x8 (*qh)[ROW / 32],
                                          const f16x8 (*ql)[ROW / 32], QX qx,
                                          const uint32_t* limit, uint32_t least, uint32_t tile,
                                          int g, int c, bool odd, KF kfrag, VF vfrag, KE kexp,
                                          VE vexp, HK k_used) {
  constexpr int KS = ROW / 32, DT = ROW / 16;
  f32x4 d[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) d[n][0] = d[n][1] = f32x4{0.f, 0.f, 0.f, 0.f};
  f16x8 k0 = kfrag(0, 0), k1 = kfrag(1, 0);
#pragma unroll
  for (int s = 0; s < KS; ++s) {  // both halves' products in turn: no MFMA waits for the last one
    f16x8 m0 = k0, m1 = k1;
    if (s + 1 < KS) k0 = kfrag(0, s + 1), k1 = kfrag(1, s + 1);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      d[n][0] = mfma16(m0, qh[n][s], d[n][0]);
      d[n][1] = mfma16(m1, qh[n][s], d[n][1]);
    }
    if constexpr (!PACK) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        d[n][0] = mfma16(m0, ql[n][s], d[n][0]);
        d[n][1] = mfma16(m1, ql[n][s], d[n][1]);
      }
    }
  }
  k_used();
  // The rare cases are branches of their own that patch what the common path
  // made (the empty asm keeps them branches, the expectation out of its way: 2 to 5% of
  // a call).
  const uint32_t key0 = tile * 32 + 4 * g;  // + r, and + 16 + r in the second half
  if constexpr (PACK) {
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int r = 0; r < 4; ++r)  // row_ror:8, the other term's column
        d[0][hh][r] += dpp_f32<0x128>(d[0][hh][r]);
  }
  auto sees = [&](int n, int i) { return key0 + (i & 3) + (i >> 2) * 16 < limit[n]; };
  float qe[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) qe[n] = ldexpf(1.f, qx(n));
  int plain = -1;  // 0: K's exponents are applied already
  if (__builtin_expect(odd, 0)) {
    asm volatile("");
    int high = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = kexp(i >> 2)[i & 3];
      high = max(high, vexp(i >> 2)[i & 3]);
#pragma unroll
      for (int n = 0; n < NT; ++n)
        d[n][i >> 2][i & 3] = e == kNanExp ? __int_as_float(0x7FC00000)
                                           : ldexpf(d[n][i >> 2][i & 3], e + qx(n));
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) qe[n] = 1.f;
    plain = 0;
    if (__builtin_expect(__any(high >= kBigExp), 0)) st.apart = true;
  }
  float w[NT][8], add[NT];
  auto weights = [&](auto masked) {
#pragma unroll
    for (int n = 0; n < NT; ++n) add[n] = 0.f;
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const i32x4 ke = kexp(hh) & plain, ve = vexp(hh);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float p =
              __builtin_amdgcn_exp2f(fmaf(ldexpf(d[n][hh][r], ke[r]), qe[n], -st.mt[n]));
          if constexpr (decltype(masked)::value) p = sees(n, 4 * hh + r) ? p : 0.f;
          add[n] += p;
          w[n][4 * hh + r] = ldexpf(p, ve[r]);
        }
    }
  };
  auto weights_apart = [&]() {
    if (__builtin_expect(st.apart, 0)) {
      asm volatile("");
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float x = ldexpf(d[n][i >> 2][i & 3], kexp(i >> 2)[i & 3] & plain);
          const float p = __builtin_amdgcn_exp2f(fmaf(x, qe[n], -st.mt[n]) +
                                                 ((float)vexp(i >> 2)[i & 3] - st.ev[n]));
          w[n][i] = sees(n, i) ? p : 0.f;
        }
    }
  };
  bool over = st.fresh;
  if (!st.fresh) {
    if (tile * 32 + 32 > least) {
      asm volatile("");
      weights(std::true_type{});
    } else {
      weights(std::false_type{});
    }
    weights_apart();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float big = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) big = fmaxf(big, w[n][i]);
      over |= big > (PACK ? 61440.f : 0x1p15f) || add[n] > 0x1p96f;
    }
  }
  if (__any(over)) {
    // New levels, of the keys that a row sees: with base the tile's largest score or the level
    // before if that is higher, the largest w next to 2^base, in (2^(r - 5), 2^(r - 4)], at 2^-4.
    asm volatile("");
    float base[NT], r[NT];
    bool far = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float x[8], mx = -INFINITY, mw = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = ldexpf(d[n][i >> 2][i & 3], kexp(i >> 2)[i & 3] & plain) * qe[n];
        x[i] = sees(n, i) ? x[i] : -INFINITY;
        mx = fmaxf(mx, x[i]);
      }
      base[n] = fmaxf(st.fresh ? -INFINITY : st.mt[n], ceilf(xor_max<32>(xor_max<16>(mx))));
      if (base[n] == -INFINITY) base[n] = 0.f;  // no key yet
#pragma unroll
      for (int i = 0; i < 8; ++i)
        mw = fmaxf(mw, (x[i] - base[n]) + (float)vexp(i >> 2)[i & 3]);
      r[n] = ceilf(xor_max<32>(xor_max<16>(mw))) + 4.f;
      if (!st.fresh) r[n] = fmaxf(r[n], (st.mt[n] - base[n]) + st.ev[n]);
      if (r[n] == -INFINITY) r[n] = 0.f;
      // One level for both, base + r: 2^30 sums of up to 2^90 stay in f32, and next to a large
      // score it may not be a 32-bit number.
      far |= r[n] < -90.f || (base[n] + r[n]) - base[n] != r[n];
      __builtin_amdgcn_sched_barrier(0);  // a row's numbers at a time: registers
    }
    if (__builtin_expect(__any(far), 0)) st.apart = true;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float m1 = st.apart ? base[n] : base[n] + r[n], e1 = st.apart ? r[n] : 0.f;
      if (!st.fresh) {
        const float by = st.mt[n] - m1;
        st.l[n] *= __builtin_amdgcn_exp2f(by);
        const float keep = __builtin_amdgcn_exp2f(by + (st.ev[n] - e1));
#pragma unroll
        for (int j = 0; j < DT; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) st.acc[n][j][i] *= keep;
      }
      st.mt[n] = m1;
      st.ev[n] = e1;
    }
    st.fresh = false;
    weights(std::true_type{});
    weights_apart();
  }
  if (__builtin_expect(odd, 0)) {
    // A row that sees a NaN row of V becomes NaN (K's made its scores NaN).
    asm volatile("");
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n)
        if (vexp(i >> 2)[i & 3] == kNanExp && sees(n, i)) w[n][i] = __int_as_float(0x7FC00000);
  }
  // The weights as B operands: hi and lo, or (PACK) the one of the lane's column.
  f16x8 ph[NT], pl[PACK ? 1 : NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    uint32_t h[4], o[4];
    st.l[n] += add[n];
    if constexpr (PACK) {
      const float mine = c < 8 ? 1.f : 2048.f, hi = c < 8 ? 0.f : -2048.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // w, or 2^11 (w - hi)
        const float x = w[n][2 * i], y = w[n][2 * i + 1];
        const h2 r = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(x, y));
        h[i] = __builtin_bit_cast(
            uint32_t, __builtin_amdgcn_cvt_pkrtz(fmaf(x, mine, (float)r[0] * hi),
                                                 fmaf(y, mine, (float)r[1] * hi)));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) split2_up(w[n][2 * i], w[n][2 * i + 1], h[i], o[i]);
      pl[n] = f16x8_of(make_uint4(o[0], o[1], o[2], o[3]));
    }
    ph[n] = f16x8_of(make_uint4(h[0], h[1], h[2], h[3]));
  }
  // O^T += V^T P^T.
  f16x8 v0 = vfrag(0), v1 = vfrag(1);
#pragma unroll
  for (int j = 0; j < DT; j += 2) {
    const f16x8 m0 = v0, m1 = v1;
    if (j + 2 < DT) v0 = vfrag(j + 2), v1 = vfrag(j + 3);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      st.acc[n][j] = mfma16(m0, ph[n], st.acc[n][j]);
      st.acc[n][j + 1] = mfma16(m1, ph[n], st.acc[n][j + 1]);
    }
    if constexpr (!PACK) {
      const f16x8 s0 = m0 * (_Float16)0x1p-11f, s1 = m1 * (_Float16)0x1p-11f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        st.acc[n][j] = mfma16(s0, pl[n], st.acc[n][j]);
        st.acc[n][j + 1] = mfma16(s1, pl[n], st.acc[n][j + 1]);
      }
    }
  }
}

// Byte J of the lane's eight keys as an A operand of V.
template <int J>
__device__ __forceinline__ f16x8 v_frag(const uint32_t* v, int stride) {
  return f16x8_of(make_uint4(pair_f16<J>(v[0], v[stride]), pair_f16<J>(v[2 * stride], v[3 * stride]),
                             pair_f16<J>(v[4 * stride], v[5 * stride]),
                             pair_f16<J>(v[6 * stride], v[7 * stride])));
}
__device__ __forceinline__ f16x8 v_frag(const uint32_t* v, int stride, int j) {
  switch (j & 3) {
    case 0: return v_frag<0>(v, stride);
    case 1: return v_frag<1>(v, stride);
    case 2: return v_frag<2>(v, stride);
    default: return v_frag<3>(v, stride);
  }
}

__device__ __forceinline__ uint64_t shfl_u64(uint64_t x, int lane) {
  return (uint64_t)(uint32_t)__shfl((int)(x >> 32), lane, 64) << 32 |
         (uint32_t)__shfl((int)(uint32_t)x, lane, 64);
}

// Four columns of a row's output, as many as the head has.
__device__ __forceinline__ uint64_t out_at(const AttnQ8Args& a, const RowRef& x) {
  return x.bt * a.out_stride + (size_t)x.head * a.c.head_dim;
}
__device__ __forceinline__ void store_out(const AttnQ8Args& a, uint64_t at, uint32_t col,
                                          f32x4 v) {
  const uint32_t hd = a.c.head_dim;
  float* out = a.out + at + col;
  if (a.out_vec) {
    if (col < hd) *reinterpret_cast<f32x4*>(out) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (col + i < hd) out[i] = v[i];
  }
}

// SHARED: the prefix's keys for the rows of all sequences, as partial results.
// Otherwise a sequence's own keys; with one split (and the prefix's partial
// results, where there are) the block writes the output itself.
//
// Straight from memory into the operands: no LDS between, since a tile is read
// by one wave.  64 sequences over 2040 keys of 16 heads of 128 (539 MB) take 87 us,
// 6.2 TB/s: the memory.  3 sequences over 84163 to 100001 keys of
// 4 heads (42 splits each) take 52 us and 5.5 for the join.  32 sequences over
// up to 511 keys of 12 heads of 64 take 6 us with warm caches and 10 without: the launch, three
// memory latencies (lengths, codes, output) and 0.85 us a tile, of which
// there are four in a row a wave.  Blocks of 8 waves take 12.6 us there in place of 10.1 (their
// registers leave room for one on a CU), but 6.9 in place of 7.4 where blocks are few (one sequence of 301
// keys); 4 waves a SIMD at 128 registers spilled, and loading a wave's second tile too before the
// lengths are known was slower (10.6 -> 11.1).
template <int ROW, bool PACK, int WAVES, bool SHARED, bool STREAM>
__global__ __launch_bounds__(64 * WAVES, ROW == 64 ? 3 : 2) void k_attn_q8(AttnQ8Args a, AttnQ8Plan pl) {
  constexpr int KS = ROW / 32;       // MFMA steps of a score
  constexpr int DT = ROW / 16;       // MFMAs of 16 output columns
  constexpr int RT = PACK ? 8 : 16;  // rows of a job
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;
  Job<SHARED> job;
  job.init(a, pl);
  const uint32_t row0 = job.group * RT;
  const Q8Cache& src = SHARED ? a.pre : a.c;
  const size_t base = ((size_t)job.b * src.kv_heads + job.kvh) * src.cap;
  const int8_t* kp = src.k + base * ROW;
  const int8_t* vp = src.v + base * ROW;
  const int8_t* kep = src.ke + base;
  const int8_t* vep = src.ve + base;

  // With one split the first tile (inside the cache wherever the rows end) is
  // under way before the lengths have arrived.
  Tile<ROW> even, odd;  // the wave's tiles in turn
  const bool early = job.splits == 1;
  if (early) {
    const uint32_t key = min((uint32_t)wave * 32, src.cap - 32);
    load_k<ROW, STREAM>(even, kp, kep, vep, key, g, c);
    load_v<ROW, STREAM>(even, vp, key, g, c);
  }
  // The prefix's parts of the job's rows, 64 WAVES / RT lanes to a row.
  constexpr int L = 64 * WAVES / RT;
  constexpr int MAXP = SHARED ? 0 : kAttnMaxSplits, NP = (MAXP + L - 1) / L;
  const bool final = !SHARED && pl.own_splits == 1;
  const uint32_t extra = final ? pl.prefix_splits : 0;
  PartMl* ml = reinterpret_cast<PartMl*>(a.ws);
  float* po = reinterpret_cast<float*>(static_cast<char*>(a.ws) + pl.rows_offset);
  const uint32_t nparts = pl.prefix_splits + (pl.own_splits > 1 ? pl.own_splits : 0);
  const int jrow = threadIdx.x / L, jl = threadIdx.x % L;
  PartMl pre[NP > 0 ? NP : 1];
  if (NP > 0 && extra) {
    const RowRef x = job.row(a, row0 + jrow);
#pragma unroll
    for (int i = 0; i < NP; ++i)
      pre[i] = x.live && jl + i * L < (int)extra ? ml[row_id(a, x) * nparts + jl + i * L]
                                                 : PartMl{-INFINITY, 0.f};
  } else {
#pragma unroll
    for (int i = 0; i < NP; ++i) pre[i] = {-INFINITY, 0.f};
  }
  // Wave 0 makes the rows' operands for all.
  __shared__ uint4 sq[PACK ? 1 : 2][KS][64];
  __shared__ int sqx[16];
  const RowRef ref = job.row(a, row0 + (PACK ? c & 7 : c));
  if (wave == 0) {
    RawQ<ROW> raw;
    raw.load(a, ref, g);
    f16x8 hi[KS], lo[KS];
    const int qe = raw.operands(a, hi, lo);
    if (g == 0) sqx[c] = qe;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      sq[0][s][lane] = __builtin_bit_cast(uint4, PACK && c >= 8 ? lo[s] : hi[s]);
      if constexpr (!PACK) sq[1][s][lane] = __builtin_bit_cast(uint4, lo[s]);
    }
  }
  // The split's tiles [t0, t1), the waves' in turn.
  uint32_t least, most;
  job.span(a, row0, RT, least, most);
  const uint32_t tiles = (most + 31) / 32;
  const uint32_t per = early ? tiles : (tiles + job.splits - 1) / job.splits;
  const uint32_t t0 = min(tiles, job.split * per), t1 = min(tiles, t0 + per);
  uint32_t t = t0 + wave;
  if (!early && t < t1) {
    load_k<ROW, STREAM>(even, kp, kep, vep, t * 32, g, c);
    load_v<ROW, STREAM>(even, vp, t * 32, g, c);
  }
  if (t + WAVES < t1) {
    load_k<ROW, STREAM>(odd, kp, kep, vep, (t + WAVES) * 32, g, c);
    load_v<ROW, STREAM>(odd, vp, (t + WAVES) * 32, g, c);
  }
  __syncthreads();
  f16x8 qh[1][KS], ql[1][KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    qh[0][s] = f16x8_of(sq[0][s][lane]);
    if constexpr (!PACK) ql[0][s] = f16x8_of(sq[1][s][lane]);
  }
  const int qx = ref.live ? sqx[c] : kNoRow;
  const bool far = __any(outside_f32(qx));
  RowsState<ROW, 1> st;
  st.init();
  auto step = [&](Tile<ROW>& tile) {
    uint32_t ke[2] = {tile.ke[0], tile.ke[1]}, ve[2] = {tile.ve[0], tile.ve[1]};
    if (t * 32 + 32 > most) {  // behind the rows' last key the exponents may be anything
      asm volatile("");
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const uint32_t key = t * 32 + 16 * hh + 4 * g;
        const int left = (int)min(most, key + 4) - (int)key;
        const uint32_t keep = left <= 0 ? 0u : 0xFFFFFFFFu >> (32 - 8 * left);
        ke[hh] &= keep;
        ve[hh] &= keep;
      }
    }
    const i32x4 e0 = exps_of(ke[0]), e1 = exps_of(ke[1]), f0 = exps_of(ve[0]), f1 = exps_of(ve[1]);
    int low = 0, high = 0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      low = min(low, min(min(e0[r], e1[r]), min(f0[r], f1[r])));
      high = max(high, max(max(e0[r], e1[r]), max(f0[r], f1[r])));
    }
    const bool more = t + 2 * WAVES < t1;
    tile_step<ROW, 1, PACK>(
        st, qh, ql, [&](int) { return qx; }, &ref.limit, least, t, g, c,
        far || __any(low == kNanExp || high >= kBigExp),
        [&](int hh, int s) {
          const uint4 w = tile.k[hh][s >> 1];
          return (s & 1) ? codes8_f16(w.z, w.w) : codes8_f16(w.x, w.y);
        },
        [&](int j) { return v_frag(&tile.v[0][j / 4], ROW / 64, j); },
        [&](int hh) { return hh ? e1 : e0; }, [&](int hh) { return hh ? f1 : f0; },
        [&]() {  // its registers take the wave's next tile but one
          if (more) load_k<ROW, STREAM>(tile, kp, kep, vep, (t + 2 * WAVES) * 32, g, c);
        });
    if (more) load_v<ROW, STREAM>(tile, vp, (t + 2 * WAVES) * 32, g, c);
    t += WAVES;
  };
  while (t < t1) {
    step(even);
    if (t >= t1) break;
    step(odd);
  }

  // Join the waves and the prefix's parts: rows normalised, weighted by sums.
  constexpr int RS = ROW + 4;
  constexpr int EL = (RT * (ROW / 4) + 64 * WAVES - 1) / (64 * WAVES);  // quads of columns a thread
  __shared__ __attribute__((aligned(16))) float so[WAVES][RT][RS];
  __shared__ PartMl sml[WAVES][RT];
  __shared__ float sw[RT][WAVES + MAXP];
  __shared__ float2 sfin[RT];  // maximum and sum of a row over all its parts
  const float total = xor_sum<32>(xor_sum<16>(st.l[0]));
  const float inv = total == 0.f ? 0.f : 1.f / total;
  const bool mine = !PACK || c < 8;
  if (g == 0 && mine) sml[wave][c] = {total == 0.f ? -INFINITY : st.mt[0], total};
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int j = 0; j < DT; j += 4) {
      f32x4 o;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[i] = st.acc[0][j + i][r];
        if constexpr (PACK) o[i] = fmaf(dpp_f32<0x128>(o[i]), 0x1p-11f, o[i]);
        o[i] *= inv;
      }
      if (__builtin_expect(st.apart, 0)) {
        asm volatile("");
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = ldexpf(o[i], (int)st.ev[0]);
      }
      if (mine && ref.live) *reinterpret_cast<f32x4*>(&so[wave][c][(4 * g + r) * DT + j]) = o;
    }
  // The thread's quads of columns, and the parts' of the first eight splits.
  const uint32_t hd = a.c.head_dim;
  const uint32_t rows_here = min((uint32_t)RT, job.nrows - row0);
  RowRef xr[EL];
  const float* pq[EL];
  f32x4 pv[EL][8];
#pragma unroll
  for (int e = 0; e < EL; ++e) {
    const uint32_t id = threadIdx.x + e * 64 * WAVES;
    xr[e] = job.row(a, row0 + id / (ROW / 4));
    xr[e].live = xr[e].live && id / (ROW / 4) < rows_here;
    pq[e] = po + row_id(a, xr[e]) * nparts * ROW + id % (ROW / 4) * 4;
    if constexpr (!SHARED) {
#pragma unroll
      for (int p = 0; p < 8; ++p)
        if (p < (int)extra && xr[e].live) pv[e][p] = *reinterpret_cast<const f32x4*>(pq[e] + p * ROW);
    }
  }
  __syncthreads();
  {
    const PartMl y = jl < WAVES ? sml[jl][jrow] : PartMl{-INFINITY, 0.f};
    float m = y.m;
#pragma unroll
    for (int i = 0; i < NP; ++i) m = fmaxf(m, pre[i].m);
    m = group_max<L>(m);
    const float f = part_sum(y, m);
    float sum = f, z[NP > 0 ? NP : 1];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      z[i] = part_sum(pre[i], m);
      sum += z[i];
    }
    sum = group_sum<L>(sum);
    const float part = sum == 0.f ? 0.f : 1.f / sum;
    if (jl < WAVES) sw[jrow][jl] = f * part;
#pragma unroll
    for (int i = 0; i < NP; ++i)
      if (jl + i * L < (int)extra) sw[jrow][WAVES + jl + i * L] = z[i] * part;
    if (jl == 0) sfin[jrow] = make_float2(m, sum);
  }
  __syncthreads();
  const uint32_t at = SHARED ? job.split : pl.prefix_splits + job.split;
#pragma unroll
  for (int e = 0; e < EL; ++e) {
    const uint32_t id = threadIdx.x + e * 64 * WAVES;
    const uint32_t row = id / (ROW / 4), col = id % (ROW / 4) * 4;
    if (row >= rows_here) continue;
    const RowRef x = xr[e];
    const float2 fin = sfin[row];
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    if (x.live) {  // (parts without a key are zeros)
#pragma unroll
      for (int w = 0; w < WAVES; ++w)
        o += sw[row][w] * *reinterpret_cast<const f32x4*>(&so[w][row][col]);
      if constexpr (!SHARED) {
#pragma unroll
        for (int p = 0; p < 8; ++p)
          if (p < (int)extra) o += sw[row][WAVES + p] * pv[e][p];
#pragma unroll 4
        for (uint32_t p = 8; p < extra; ++p)
          o += sw[row][WAVES + p] * *reinterpret_cast<const f32x4*>(pq[e] + (size_t)p * ROW);
      }
    }
    if (final) {
      store_out(a, out_at(a, x), col, o);
      if (col == 0 && a.lse)
        a.lse[row_id(a, x)] =
            x.live && fin.y != 0.f ? (fin.x + log2f(fin.y)) * 0.6931471805599453f : -INFINITY;
    } else if (x.live) {
      *reinterpret_cast<f32x4*>(po + (row_id(a, x) * nparts + at) * ROW + col) = o;
      if (col == 0) ml[row_id(a, x) * nparts + at] = {fin.y == 0.f ? -INFINITY : fin.x, fin.y};
    }
  }
}

// The same for jobs of 32 RW rows (64 or 128): the block's waves convert each stage of 64
// keys to fp16 once, into LDS in the order of the MFMAs' operands, and every wave
// takes its 32 rows (wave % RW) over one of the stage's two 32-key tiles (wave / RW) from there;
// the tiles' halves are joined at the end.  The next stage's codes are on
// their way while a stage is computed, and are converted into the other half
// of the buffer.
//
// 256 rows over 8200 keys of 16 heads of 128 take 53 us: about 10 before and after
// the loop, then 2 us a stage (1000 TFLOP/s of fp16 products, both terms of q
// and of the weights counted), more where levels move.  A stage is 1000
// cycles of MFMAs a wave and 1350 of vector operations (exponents, 2^x, splitting the
// weights, converting codes), two waves a SIMD.  Stages of 128 keys, codes two stages
// ahead, wave priorities (by half, or around the products), exponents
// fetched ahead, and levels moved by the weights' own exponents measured within 2%.
template <int ROW, int RW, bool SHARED>
__global__ __launch_bounds__(128 * RW, 2) void k_attn_q8_rows(AttnQ8Args a, AttnQ8Plan pl) {
  constexpr int KS = ROW / 32, DT = ROW / 16, NT = 2, U = ROW / 64, W = 2 * RW;
  constexpr int FRAGS = 2 * KS + DT;                  // of a tile, 1 KB each
  constexpr int NK = 4 * U, NV = 2 * U;               // conversion units of a stage
  constexpr int KU = (NK + W - 1) / W, VU = (NV + W - 1) / W;
  constexpr int RS = ROW + 4;
  constexpr size_t kBuffers = (size_t)2 * 2 * FRAGS * 64;  // in uint4
  constexpr size_t kJoin = (size_t)RW * 32 * RS / 4 + RW * 16;
  __shared__ uint4 smem[kBuffers > kJoin ? kBuffers : kJoin];
  __shared__ __attribute__((aligned(16))) int exps[2][2][64];  // a stage's exponents, K's and V's
  __shared__ uint32_t odds[2][2];  // whether its tiles are odd
  __shared__ int sqx[32 * RW];
  static_assert((size_t)W * KS * 2 * 64 <= kBuffers, "the rows' operands fit the buffers");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int rw = wave % RW, kw = wave / RW;
  Job<SHARED> job;
  job.init(a, pl);
  const Q8Cache& src = SHARED ? a.pre : a.c;
  const uint32_t row0 = job.group * 32 * RW + rw * 32;
  // The wave's rows, and as far as the block's furthest one.
  uint32_t least, mine, unused, most;
  job.span(a, row0, 32, least, mine);
  job.span(a, job.group * 32 * RW, 32 * RW, unused, most);

  const uint32_t tiles = (most + 31) / 32;
  const uint32_t per = ((tiles + 1) / 2 + job.splits - 1) / job.splits * 2;  // whole stages
  const uint32_t t0 = min(tiles, job.split * per), t1 = min(tiles, t0 + per);
  const size_t base = ((size_t)job.b * src.kv_heads + job.kvh) * src.cap;
  const int8_t* kp = src.k + base * ROW;
  const int8_t* vp = src.v + base * ROW;
  const int8_t* kep = src.ke + base;
  const int8_t* vep = src.ve + base;

  uint4 rk[KU];
  uint32_t rv[VU][8];
  int re[2] = {0, 0};  // exponents of key `lane` of the stage, the last wave's
  bool re_in = false;
  auto load = [&](uint32_t t) {  // the stage of tiles t and t + 1
#pragma unroll
    for (int i = 0; i < KU; ++i) {
      const int u = wave + i * W;
      if (u < NK) {
        const uint32_t key = min(t + u / (2 * U), t1 - 1) * 32 + u / U % 2 * 16 + c;
        rk[i] = *reinterpret_cast<const uint4*>(kp + (size_t)key * ROW + 16 * g + u % U * 64);
      }
    }
#pragma unroll
    for (int i = 0; i < VU; ++i) {
      const int u = W - 1 - wave + i * W;
      if (u < NV) {
        const uint32_t key = min(t + u / U, t1 - 1) * 32 + 4 * g;
        const int8_t* q = vp + (size_t)key * ROW + c * (ROW / 16) + u % U * 4;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          rv[i][k] = *reinterpret_cast<const uint32_t*>(q + ((k & 3) + (k >> 2) * 16) * ROW);
      }
    }
    if (wave == W - 1) {
      const uint32_t key = min(t + lane / 32, t1 - 1) * 32 + lane % 32;
      re_in = key < most;  // behind that there may be anything
      re[0] = kep[key];
      re[1] = vep[key];
    }
  };
  auto store = [&](int half) {
    uint4* to = smem + (size_t)half * 2 * FRAGS * 64 + lane;
#pragma unroll
    for (int i = 0; i < KU; ++i) {
      const int u = wave + i * W;
      if (u < NK) {
        uint4* f = to + (u / (2 * U) * FRAGS + u / U % 2 * KS + u % U * 2) * 64;
        f[0] = __builtin_bit_cast(uint4, codes8_f16(rk[i].x, rk[i].y));
        f[64] = __builtin_bit_cast(uint4, codes8_f16(rk[i].z, rk[i].w));
      }
    }
#pragma unroll
    for (int i = 0; i < VU; ++i) {
      const int u = W - 1 - wave + i * W;
      if (u < NV) {
        uint4* f = to + (u / U * FRAGS + 2 * KS + u % U * 4) * 64;
        f[0] = __builtin_bit_cast(uint4, v_frag<0>(rv[i], 1));
        f[64] = __builtin_bit_cast(uint4, v_frag<1>(rv[i], 1));
        f[128] = __builtin_bit_cast(uint4, v_frag<2>(rv[i], 1));
        f[192] = __builtin_bit_cast(uint4, v_frag<3>(rv[i], 1));
      }
    }
    if (wave == W - 1) {
      const int ek = re_in ? re[0] : 0, ev = re_in ? re[1] : 0;
      exps[half][0][lane] = ek;
      exps[half][1][lane] = ev;
      const uint64_t odd = __ballot(min(ek, ev) == kNanExp || max(ek, ev) >= kBigExp);
      if (lane < 2) odds[half][lane] = (uint32_t)(odd >> (32 * lane));
    }
  };

  if (t0 < t1) load(t0);
  // The rows' operands, 16 rows a wave: whole rows into LDS (read where the
  // operands want them, a line would be fetched eight times over), from there
  // as operands, which all the rows' waves take by way of the buffer.
  constexpr int QR = ROW / 4, RI = 64 / QR;  // quads of a row, rows of a 64-lane access
  {
    const RowRef x = job.row(a, job.group * 32 * RW + wave * 16 + c);
    const uint64_t at = x.bt * a.q_stride + (size_t)x.head * a.c.head_dim;
    const int hd = (int)a.c.head_dim, d = lane % QR * 4;
    float* own = reinterpret_cast<float*>(smem) + (size_t)wave * 16 * RS;
    f32x4 v[16 / RI];
#pragma unroll
    for (int i = 0; i < 16 / RI; ++i) {
      const float* q = a.q + shfl_u64(at, i * RI + lane / QR);
      if (a.q_vec) {
        v[i] = *reinterpret_cast<const f32x4*>(q + min(d, hd - 4));
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[i][k] = q[min(d + k, hd - 1)];
      }
    }
#pragma unroll
    for (int i = 0; i < 16 / RI; ++i) {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[i][k] = d + k < hd ? v[i][k] : 0.f;
      *reinterpret_cast<f32x4*>(own + (i * RI + lane / QR) * RS + d) = v[i];
    }
    __builtin_amdgcn_wave_barrier();  // a wave's LDS accesses keep their order
    RawQ<ROW> raw;
    raw.from_lds(own, RS, g, c);
    f16x8 hi[KS], lo[KS];
    const int qe = raw.operands(a, hi, lo);
    if (g == 0) sqx[wave * 16 + c] = x.live ? qe : kNoRow;
    __syncthreads();
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      smem[((wave * KS + s) * 2) * 64 + lane] = __builtin_bit_cast(uint4, hi[s]);
      smem[((wave * KS + s) * 2 + 1) * 64 + lane] = __builtin_bit_cast(uint4, lo[s]);
    }
  }
  RowRef ref[NT];
  uint32_t limit[NT];
  f16x8 qh[NT][KS], ql[NT][KS];
  bool far = false;
  int qx[NT];
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    ref[n] = job.row(a, row0 + n * 16 + c);
    limit[n] = ref[n].limit;
    qx[n] = sqx[rw * 32 + n * 16 + c];
    far |= __any(outside_f32(qx[n]));
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      qh[n][s] = f16x8_of(smem[(((rw * 2 + n) * KS + s) * 2) * 64 + lane]);
      ql[n][s] = f16x8_of(smem[(((rw * 2 + n) * KS + s) * 2 + 1) * 64 + lane]);
    }
  }
  __syncthreads();
  RowsState<ROW, NT> st;
  st.init();
  if (t0 < t1) store(0);
  int half = 0;
  for (uint32_t t = t0; t < t1; t += 2) {
    __syncthreads();
    if (t + 2 < t1) load(t + 2);
    if (t + kw < t1 && (t + kw) * 32 < mine) {
      const uint4* f = smem + ((size_t)half * 2 + kw) * FRAGS * 64 + lane;
      const int* e = &exps[half][0][32 * kw + 4 * g];
      tile_step<ROW, NT, false>(
          st, qh, ql, [&](int n) { return qx[n]; }, limit, least, t + kw, g, c,
          far || __builtin_amdgcn_readfirstlane(odds[half][kw]) != 0,
          [&](int hh, int s) { return f16x8_of(f[(hh * KS + s) * 64]); },
          [&](int j) { return f16x8_of(f[(2 * KS + j) * 64]); },
          [&](int hh) { return *reinterpret_cast<const i32x4*>(e + 16 * hh); },
          [&](int hh) { return *reinterpret_cast<const i32x4*>(e + 64 + 16 * hh); }, []() {});
    }
    half ^= 1;
    if (t + 2 < t1) store(half);
  }

  // The two waves of the same rows exchange 16 rows each, normalised, and
  // finish the other 16.
  __syncthreads();
  float* so = reinterpret_cast<float*>(smem);
  PartMl* sml = reinterpret_cast<PartMl*>(so + (size_t)RW * 32 * RS);
  float m[NT], total[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    total[n] = xor_sum<32>(xor_sum<16>(st.l[n]));
    m[n] = total[n] == 0.f ? -INFINITY : st.mt[n];
    const float inv = total[n] == 0.f ? 0.f : 1.f / total[n];
#pragma unroll
    for (int j = 0; j < DT; ++j) st.acc[n][j] *= inv;
    if (__builtin_expect(st.apart, 0)) {
      asm volatile("");
#pragma unroll
      for (int j = 0; j < DT; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) st.acc[n][j][r] = ldexpf(st.acc[n][j][r], (int)st.ev[n]);
    }
  }
  const int row = rw * 32 + c;  // + 16 for the rows of kw = 1
  auto hand = [&](const f32x4* acc, float mm, float ll, int r16) {
    if (g == 0) sml[row + r16] = {mm, ll};
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < DT; j += 4)
        *reinterpret_cast<f32x4*>(so + (size_t)(row + r16) * RS + (4 * g + r) * DT + j) =
            f32x4{acc[j][r], acc[j + 1][r], acc[j + 2][r], acc[j + 3][r]};
  };
  if (kw == 0)
    hand(st.acc[1], m[1], total[1], 16);
  else
    hand(st.acc[0], m[0], total[0], 0);
  __syncthreads();
  const bool final = !SHARED && pl.own_splits == 1;
  const uint32_t extra = final ? pl.prefix_splits : 0;
  PartMl* ml = reinterpret_cast<PartMl*>(a.ws);
  float* po = reinterpret_cast<float*>(static_cast<char*>(a.ws) + pl.rows_offset);
  const uint32_t nparts = pl.prefix_splits + (pl.own_splits > 1 ? pl.own_splits : 0);
  const uint32_t at = SHARED ? job.split : pl.prefix_splits + job.split;
  auto finish = [&](f32x4* acc, float mm, float ll, const RowRef& x, int r16) {
    const size_t part = row_id(a, x) * nparts;
    const PartMl y = sml[row + r16];
    float top = fmaxf(mm, y.m);
    for (uint32_t e = 0; e < extra && x.live; ++e) top = fmaxf(top, ml[part + e].m);
    const float f0 = part_sum({mm, ll}, top), f1 = part_sum(y, top);
    float sum = f0 + f1;
    for (uint32_t e = 0; e < extra && x.live; ++e) sum += part_sum(ml[part + e], top);
    const float inv = x.live && sum != 0.f ? 1.f / sum : 0.f;
    float* mine = so + (size_t)(row + r16) * RS + 4 * g * DT;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < DT; j += 4) {
        f32x4* at = reinterpret_cast<f32x4*>(mine + r * DT + j);
        *at = f0 * inv * f32x4{acc[j][r], acc[j + 1][r], acc[j + 2][r], acc[j + 3][r]} +
              f1 * inv * *at;
      }
    __builtin_amdgcn_wave_barrier();  // a wave's LDS accesses keep their order
    // Whole rows from here.
    const bool there = row0 + r16 + c < job.nrows && (x.live || final);
    const uint64_t flags = __ballot(there), lives = __ballot(x.live);
    const uint64_t o_at = out_at(a, x);
#pragma unroll
    for (int i = 0; i < 16 / RI; ++i) {
      const int r = i * RI + lane / QR, col = lane % QR * 4;
      const size_t p = shfl_u64(part, r);
      const uint64_t out = shfl_u64(o_at, r);
      f32x4 o = *reinterpret_cast<const f32x4*>(so + (size_t)(rw * 32 + r16 + r) * RS + col);
      if (extra) {
        const float t = __shfl(top, r, 64), n = __shfl(inv, r, 64);
        if (lives >> r & 1)
          for (uint32_t e = 0; e < extra; ++e)
            o += part_sum(ml[p + e], t) * n * *reinterpret_cast<const f32x4*>(po + (p + e) * ROW + col);
      }
      if (!(lives >> r & 1)) o = f32x4{0.f, 0.f, 0.f, 0.f};
      if (flags >> r & 1) {
        if (!final)
          *reinterpret_cast<f32x4*>(po + (p + at) * ROW + col) = o;
        else
          store_out(a, out, col, o);
      }
    }
    if (g == 0 && there) {
      const bool some = x.live && sum != 0.f;
      if (!final)
        ml[part + at] = {some ? top : -INFINITY, some ? sum : 0.f};
      else if (a.lse)
        a.lse[row_id(a, x)] = some ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
    }
  };
  if (kw == 0)
    finish(st.acc[0], m[0], total[0], ref[0], 0);
  else
    finish(st.acc[1], m[1], total[1], ref[1], 16);
}

// Joins a row's partial results: one block per row and head, a wave takes
// every fourth part.  48 rows of 42 parts (of 128) take 5.5 us: two memory
// latencies and the launch.
template <int ROW>
__global__ __launch_bounds__(256) void k_attn_q8_join(AttnQ8Args a, AttnQ8Plan pl) {
  constexpr int C = ROW / 64;
  const uint32_t id = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t bt = id / a.heads;
  const uint32_t b = bt / a.rows, t = bt % a.rows;
  float* out = a.out + (size_t)bt * a.out_stride + (size_t)(id % a.heads) * a.c.head_dim;
  const int n = pl.prefix_splits + pl.own_splits;  // at most two a lane
  const PartMl* ml = reinterpret_cast<const PartMl*>(a.ws) + (size_t)id * n;
  const float* po =
      reinterpret_cast<const float*>(static_cast<const char*>(a.ws) + pl.rows_offset) +
      (size_t)id * n * ROW + lane;
  __shared__ float part[4][ROW];
  float m = -INFINITY, total = 0.f, o[C] = {};
  if (t < step_rows(a.counts, b, a.rows)) {
    PartMl y[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      y[i] = lane + 64 * i < n ? ml[lane + 64 * i] : PartMl{-INFINITY, 0.f};
    m = wave_max(fmaxf(y[0].m, y[1].m));
    float f[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) f[i] = part_sum(y[i], m);
    total = wave_sum(f[0] + f[1]);
    const float inv = total == 0.f ? 0.f : 1.f / total;
    f[0] *= inv;
    f[1] *= inv;
    for (int p = wave; p < n; p += 4) {
      const float w = __shfl(p < 64 ? f[0] : f[1], p & 63, 64);
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const float x = po[(size_t)p * ROW + 64 * i];
        o[i] += w * x;  // (a part without a key is zeros)
      }
    }
  }
#pragma unroll
  for (int i = 0; i < C; ++i) part[wave][lane + 64 * i] = o[i];
  __syncthreads();
  const uint32_t col = threadIdx.x;
  if (col < a.c.head_dim)
    out[col] = ((part[0][col] + part[1][col]) + part[2][col]) + part[3][col];
  if (threadIdx.x == 0 && a.lse)
    a.lse[id] = total == 0.f ? -INFINITY : (m + log2f(total)) * 0.6931471805599453f;
}

uint64_t div_up(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

bool vec4(const void* p, uint32_t stride, uint32_t head_dim) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % 4 == 0 && head_dim % 4 == 0;
}

}  // namespace

namespace {

// One row a thread for a decode step's, four for longer stretches.
Q8Rows rows_of(const Q8Cache& c, uint32_t batch, uint32_t rows, uint32_t stride,
               const uint32_t* pos, const uint32_t* counts, uint32_t r, uint64_t* blocks) {
  Q8Rows a{batch, rows, stride, (uint32_t)div_up(rows, r),
           (uint32_t)div_up(2 * (uint64_t)c.kv_heads, 1024 / c.row), pos, counts};
  *blocks = (uint64_t)batch * a.groups * a.blocks;
  return a;
}

}  // namespace

uint64_t cache_q8_blocks(const Q8Cache& c, uint32_t batch, uint32_t rows) {
  uint64_t blocks;
  rows_of(c, batch, rows, 0, nullptr, nullptr, rows > 1 ? 4 : 1, &blocks);
  return blocks;
}

hipError_t launch_cache_write_q8(const float* k, const float* v, const Q8Cache& c, uint32_t batch,
                                 uint32_t rows, uint32_t stride, const uint32_t* pos,
                                 const uint32_t* counts, hipStream_t s) {
  const bool vec = vec4(k, stride, c.head_dim) && vec4(v, stride, c.head_dim);
  const bool many = rows > 1;
  uint64_t blocks;
  const Q8Rows a = rows_of(c, batch, rows, stride, pos, counts, many ? 4 : 1, &blocks);
#define AKH_PICK(F, ROW)                                               \
  (many ? (vec ? F<ROW, 4, true> : F<ROW, 4, false>)                   \
        : (vec ? F<ROW, 1, true> : F<ROW, 1, false>))
  auto* f = c.row == 128 ? AKH_PICK(k_cache_write_q8, 128) : AKH_PICK(k_cache_write_q8, 64);
  hipLaunchKernelGGL(f, dim3((uint32_t)blocks), dim3(256), 0, s, k, v, c, a);
  return hipGetLastError();
}

hipError_t launch_cache_read_q8(const Q8Cache& c, float* k, float* v, uint32_t batch,
                                uint32_t rows, uint32_t stride, const uint32_t* pos,
                                const uint32_t* counts, hipStream_t s) {
  const bool vec = (!k || vec4(k, stride, c.head_dim)) && (!v || vec4(v, stride, c.head_dim));
  const bool many = rows > 1;
  uint64_t blocks;
  const Q8Rows a = rows_of(c, batch, rows, stride, pos, counts, many ? 4 : 1, &blocks);
  auto* f = c.row == 128 ? AKH_PICK(k_cache_read_q8, 128) : AKH_PICK(k_cache_read_q8, 64);
#undef AKH_PICK
  hipLaunchKernelGGL(f, dim3((uint32_t)blocks), dim3(256), 0, s, c, k, v, a);
  return hipGetLastError();
}

namespace {

constexpr uint64_t kCus = 256;

// How `jobs` (kv heads of sequences, or of the prefix) of `rows` query rows
// each and `tiles` 32-key tiles are dealt: rows of a block (8 in packed
// columns, 16, or 64 and 128 by way of LDS), its waves, and splits of the
// keys, from a model of the time in us.  Direct blocks: 4.5 or 5 us (2 more where
// CUs get a second one), and each of a wave's tiles 0.85 alone; with the CUs full (8
// waves of 128 columns, 12 of 64) 1.65 or 2, or 2.75 where the codes come from
// memory and no other group reads them.  Blocks in LDS: 8 of their waves on a
// CU, 7 or 8.5 us and 1.4 to 2.8 or 2.1 a stage of 64 keys.  Splits cost a join, and
// their rows written and read.  Over 72 shapes drawn from 1 to 256 rows and 64 to
// 30000 keys the choice's time is 0.9% above the fastest kind's of rows per block, 16% at
// the worst (profiles/q8_plan_shapes.md); taking the largest block that the rows fill was up to
// 2 times it (16 x 20 rows of 12 heads over 2, 400 keys: 17.8 us, here 8.5).
struct Deal {
  uint32_t rt, groups, waves, splits;
};
Deal deal(uint64_t jobs, uint64_t rows, uint64_t tiles, uint32_t row, uint64_t ids, bool joined) {
  static const uint32_t kSplits[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 21, 25, 32, 42, 51, 64};
  Deal best{};
  double least = 1e300;
  for (uint32_t rt : {8u, 16u, 64u, 128u}) {
    if (rt > 8 && rt / 2 >= rows && rt != 64) break;
    if (rt == 64 && rows <= 16) break;
    const bool direct = rt <= 16;
    const uint64_t groups = div_up(rows, rt), blocks = jobs * groups;
    const double cap = (double)kCus * (direct && row == 64 ? 12 : 8);
    const double shared = std::max(rt == 8 ? 0.8 : 1.15, 1.9 / (double)groups);
    const uint32_t most = direct ? 4 : rt / 16;
    for (uint32_t w = rt == 8 ? 2 : most; w <= most; w += 2)  // (2 waves of 16 rows spill)
      for (uint32_t s : kSplits) {
        if (s > 1 && (s > kAttnMaxSplits || blocks * s * w > kMaxBlocks * 4 ||
                      tiles / s < (direct ? 2 * w : 4)))
          break;
        const double full = (double)(blocks * s * w) / cap;
        const double rounds = full <= 1 ? 1 : full <= 4 ? (double)(uint64_t)(full + 0.999) : full;
        const double at_once = full < 1 ? full : 1;
        const double second = std::min(std::max((double)(blocks * s * w) / (4 * kCus) - 1, 0.0), 1.0);
        double t = direct ? (rt == 8 ? 4.5 : 5) + 2 * second + (double)div_up(tiles, (uint64_t)s * w) *
                                                      (0.85 + shared * at_once)
                   : rt == 64 ? 7 + (double)div_up(tiles, 2 * (uint64_t)s) * (1.4 + 1.4 * at_once)
                              : 8.5 + (double)div_up(tiles, 2 * (uint64_t)s) * 2.1;
        t *= rounds;
        if (s > 1 || joined) t += (double)ids * s * row * 8 / 6e6;
        if (s > 1 && !joined) t += 4;
        if (w == 2) t *= 1.05;  // four waves even out a block's tail
        if (t < least) {
          least = t;
          best = {rt, (uint32_t)groups, w, s};
        }
      }
  }
  return best;
}

AttnQ8Plan attn_q8_plan(const AttnQ8Args& a, bool prefix) {
  AttnQ8Plan p{};
  const uint64_t G = a.heads / a.c.kv_heads;
  p.G = (uint32_t)G;
  const uint64_t own = a.rows * G, all = own * a.batch;
  const uint64_t ids = (uint64_t)a.batch * a.rows * a.heads;
  const Deal d = deal((uint64_t)a.batch * a.c.kv_heads, own, div_up(a.max_len, 32), a.c.row, ids,
                      false);
  p.own_rt = d.rt;
  p.own_groups = d.groups;
  p.own_splits = d.splits;
  p.own_waves = d.waves;
  // Caches that the 256 MB behind the L2s will not hold until they are read
  // again: 64 sequences x 16 heads of 128, us with and without streaming:
  // 256 rows (68 MB) 17.2 and 15.9, 512 27.9 and 30.2, 2048 88.3 and 96.7.  Not with several
  // groups of query rows, which read the same codes by way of one L2: 64 x 20 rows over 2048 keys
  // of 16 heads of 128 (2 groups) 179 and 157, 1 x 9 rows of 16 heads over 120000 keys of 4 heads of
  // 128 (3 groups) 62.2 and 56.3, 64 x 24 rows over 2048 keys of 12 heads of 64 (2) 72.6 and 70.2.
  p.stream = p.own_groups == 1 && (uint64_t)a.batch * a.c.kv_heads *
                                      a.max_len * 2 * a.c.row > (96ull << 20);
  if (prefix) {  // its parts are joined with the own rows' in any case
    const Deal e = deal(a.c.kv_heads, all, div_up(a.pre.max_rows, 32), a.c.row, ids, true);
    p.prefix_rt = e.rt;
    p.prefix_groups = e.groups;
    p.prefix_splits = e.splits;
    p.prefix_waves = e.waves;
  }
  const uint64_t parts = p.prefix_splits + (p.own_splits > 1 ? p.own_splits : 0);
  p.rows_offset = div_up(ids * parts * sizeof(PartMl), 16) * 16;
  p.bytes = parts ? p.rows_offset + ids * parts * a.c.row * sizeof(float) : 0;
  return p;
}

template <int ROW, bool SHARED>
void launch_parts(const AttnQ8Args& a, const AttnQ8Plan& p, hipStream_t s) {
  const uint32_t rt = SHARED ? p.prefix_rt : p.own_rt;
  const dim3 grid(SHARED ? p.prefix_groups * a.c.kv_heads * p.prefix_splits
                         : a.batch * p.own_splits * a.c.kv_heads * p.own_groups);
  const uint32_t waves = SHARED ? p.prefix_waves : p.own_waves;
  auto direct = [&](auto pack) {
    constexpr bool PACK = decltype(pack)::value;
    constexpr int FEW = PACK ? 2 : 4;
    if constexpr (!SHARED)
      if (p.stream)
        return waves == 2 ? k_attn_q8<ROW, PACK, FEW, false, true> : k_attn_q8<ROW, PACK, 4, false, true>;
    return waves == 2 ? k_attn_q8<ROW, PACK, FEW, SHARED, false> : k_attn_q8<ROW, PACK, 4, SHARED, false>;
  };
  auto* f = rt == 8    ? direct(std::true_type{})
            : rt == 16 ? direct(std::false_type{})
            : rt == 64 ? k_attn_q8_rows<ROW, 2, SHARED>
                       : k_attn_q8_rows<ROW, 4, SHARED>;
  const uint32_t threads = waves * 64;
  hipLaunchKernelGGL(f, grid, dim3(threads), 0, s, a, p);
}

template <int ROW>
hipError_t launch_attn(const AttnQ8Args& a, const AttnQ8Plan& p, hipStream_t s) {
  if (p.prefix_splits) launch_parts<ROW, true>(a, p, s);
  launch_parts<ROW, false>(a, p, s);
  if (p.own_splits > 1)
    hipLaunchKernelGGL((k_attn_q8_join<ROW>), dim3(a.batch * a.rows * a.heads), dim3(256), 0, s, a,
                       p);
  return hipGetLastError();
}

}  // namespace

size_t attn_q8_workspace_bytes(const AttnQ8Args& a, bool prefix) {
  return a.batch && a.rows ? attn_q8_plan(a, prefix).bytes : 0;
}

hipError_t launch_attn_q8(AttnQ8Args a, hipStream_t s) {
  const AttnQ8Plan p = attn_q8_plan(a, a.prefix_len != nullptr);
  a.scale_mant = (float)std::frexp((double)a.scale * 1.4426950408889634, &a.scale_exp);
  a.q_vec = vec4(a.q, a.q_stride, a.c.head_dim);
  a.out_vec = vec4(a.out, a.out_stride, a.c.head_dim);
  return a.c.row == 128 ? launch_attn<128>(a, p, s) : launch_attn<64>(a, p, s);
}

}  // namespace akh
