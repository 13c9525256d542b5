// Attention over view tokens, forward and backward, for 16-bit tensors:
//   S = scale q k^T over the kept keys,  P = exp(S - lse),  O = P v
//   dV = P^T dO,  dS = P (dO v^T - delta),  delta = rowsum(dO O),  dQ = scale dS k,  dK = scale dS^T q
// One pass over the keys with the running maximum and sum; nothing of size queries x keys is ever stored: the backward recomputes the
// probabilities from q, k and lse.  Sums, maxima and exponentials are 32 bits wide; P and dS are rounded to the tensors' type where they
// enter a matrix instruction (P lies in [0, 1] and dS enters as a factor: half a step of the type relative to each, as of the inputs).
//
// All three kernels have one shape.  A wave owns 32 columns — queries (forward, dQ) or keys (dK/dV) — and walks the other side in tiles that its
// workgroup stages in LDS.  Scores come as tile x columns from v_mfma_f32_32x32x16: a lane then holds 16 scores of ONE column (rows 8 (r / 4) +
// 4 (lane / 32) + r % 4), so softmax statistics need one exchange between the wave's halves, and eight consecutive registers are, with the
// tile's rows taken in that same order, an operand of the next product: probabilities never leave the registers.  The other operand of
// that product is the tile's transpose, which ds_read_b64_tr_b16 reads from the row-major tile.
//
// Key/value heads shared by several heads: the rows of the group's heads are taken as one long list (head by head), so a tile of k and v is
// staged once for all of them and dK, dV are summed in registers.  dQ and dK/dV are two kernels (7 products in place of 5) so that no sum
// depends on the order of atomics: gradients repeat bit by bit, as the renderer's do.
#include <math.h>

#include "mvr_token_types.h"

using namespace mvr_tok;

namespace {

constexpr int kBlock = 256, kWaves = 4;
constexpr int kTile = 64;        // rows of a staged tile

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
template <typename T> struct Vec;
template <> struct Vec<bf16> { typedef bf16x8 type; };
template <> struct Vec<f16> { typedef f16x8 type; };

__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

struct AttArgs {
  const void *q, *k, *v, *o, *go;
  const uint8_t *keep;
  void *out, *dq, *dk, *dv;
  float *lse;                    // (B, heads, queries): log2 of the sum of exp2(scale log2(e) q k); +inf for a row without keys
  float *delta;                  // the same shape
  float *part, *part_lse;        // splits over the keys: (splits, B kv_heads rows, D) and (splits, B kv_heads rows)
  int64_t qs[3], ks[3], vs[3], gs[3];
  int32_t B, Lq, Lk, H, E, G, D;   // E: kv heads, G: heads of a group
  int32_t groups, per;           // keep: (B, groups), `per` keys each
  int32_t rows;                  // G * Lq
  int32_t tiles, splits, split_tiles, col_tiles;
  int64_t work;                  // workgroups with something to do
  float c, scale;                // scale log2(e)
};

// Workgroups are dealt to the 8 XCDs round robin: item = a contiguous run of the work per XCD, so that the workgroups which read one
// object's keys share an L2
__device__ __forceinline__ int64_t work_item(int64_t work) {
  const int64_t per = (work + 7) / 8;
  return (int64_t)(blockIdx.x % 8) * per + blockIdx.x / 8;
}

template <typename T>
__device__ __forceinline__ u32x4 load16(const T *p, int left) {
  u32x4 r = {0, 0, 0, 0};
  if (left >= 8) {
    __builtin_memcpy(&r, p, 16);
  } else if (left > 0) {
    T t[8] = {};
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < left) t[k] = p[k];
    __builtin_memcpy(&r, t, 16);
  }
  return r;
}

// A tile of kTile rows on its way from memory to LDS; `row` gives a row's address, or null for a row of zeros
template <typename T, int DP>
struct Stage {
  static constexpr int kChunks = kTile * DP / 8 / kBlock, kPitch = DP + 8;
  u32x4 r[kChunks];
  template <typename Row>
  __device__ __forceinline__ void load(int D, Row row) {
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const int e = threadIdx.x + k * kBlock, i = e / (DP / 8), c = e % (DP / 8) * 8;
      const T *p = row(i);
      r[k] = load16(p + c, p ? D - c : 0);
    }
  }
  __device__ __forceinline__ void store(T *lds) const {
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const int e = threadIdx.x + k * kBlock, i = e / (DP / 8), c = e % (DP / 8) * 8;
      *reinterpret_cast<u32x4 *>(lds + i * kPitch + c) = r[k];
    }
  }
};

// operand with the tile's rows 32 t + (lane % 32) as its rows, d = 16 s + 8 (lane / 32) + 0..7 as its depth
template <typename T, int DP>
__device__ __forceinline__ typename Vec<T>::type row_frag(const T *lds, int t, int s) {
  const int lane = threadIdx.x & 63;
  return *reinterpret_cast<const typename Vec<T>::type *>(lds + (32 * t + (lane & 31)) * (DP + 8) + 16 * s + 8 * (lane >> 5));
}
// operand with d = 32 db + (lane % 32) as its rows, the tile's rows 16 s + 4 (lane / 32) + {0..3, 8..11} as its depth
template <typename T, int DP>
__device__ __forceinline__ typename Vec<T>::type col_frag(const T *lds, int s, int db) {
  typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
  const int lane = threadIdx.x & 63;
  const T *p = lds + (16 * s + 4 * (lane >> 5) + ((lane & 15) >> 2)) * (DP + 8) + 32 * db + (lane & 16) + 4 * (lane & 3);
  union { i16x4 h[2]; typename Vec<T>::type v; } u;
  u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)p);
  u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(p + 8 * (DP + 8)));
  return u.v;
}
template <typename T>
__device__ __forceinline__ typename Vec<T>::type to_frag(const f32x16 &x, int half) {
  typename Vec<T>::type v;
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = (T)x[8 * half + k];
  return v;
}
// rows of a tensor straight into operands: this lane's row p (null: zeros)
template <typename T, int DP>
__device__ __forceinline__ void load_frags(const T *p, int D, typename Vec<T>::type (&f)[DP / 16]) {
  const int hi = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const u32x4 r = load16(p + 16 * s + 8 * hi, p ? D - 16 * s - 8 * hi : 0);
    __builtin_memcpy(&f[s], &r, 16);
  }
}

// which of a tile's keys are there, one bit each
__device__ __forceinline__ unsigned long long tile_keys(const AttArgs &a, int b, int tile) {
  const int key = tile * kTile + (threadIdx.x & 63);
  bool on = key < a.Lk;
  if (a.keep && on) on = a.keep[(int64_t)b * a.groups + key / a.per] != 0;
  return __ballot(on);
}

// Walks the tiles [first, last) of one object that hold a kept key; step(tile, keys) is called by all waves alike
template <typename Load, typename Store, typename Step>
__device__ __forceinline__ void walk_tiles(const AttArgs &a, int b, int first, int last, Load load, Store store, Step step) {
  __shared__ unsigned long long masks[64];
  const int wave = threadIdx.x >> 6;
  for (int c0 = first; c0 < last; c0 += 64) {
    const int n = last - c0 < 64 ? last - c0 : 64;
    lds_barrier();   // the previous chunk's masks and tiles have been read
    for (int i = wave; i < n; i += kWaves) {
      const unsigned long long m = tile_keys(a, b, c0 + i);
      if ((threadIdx.x & 63) == 0) masks[i] = m;
    }
    lds_barrier();
    int i = 0;
    while (i < n && !masks[i]) ++i;
    unsigned long long m = i < n ? masks[i] : 0;
    if (i < n) load(c0 + i, m);
    while (i < n) {
      lds_barrier();
      store();
      lds_barrier();
      int next = i + 1;
      while (next < n && !masks[next]) ++next;
      const unsigned long long mn = next < n ? masks[next] : 0;
      if (next < n) load(c0 + next, mn);
      step(c0 + i, m);
      i = next, m = mn;
    }
  }
}

__device__ __forceinline__ unsigned long long uniform(unsigned long long m) {
  return (unsigned long long)__builtin_amdgcn_readfirstlane((int)(m >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)m);
}

// ---- forward -----------------------------------------------------------------------------------------------------

template <typename T, int DP, bool SPLIT>
__global__ __launch_bounds__(kBlock, 2) void k_attend(AttArgs a) {
  typedef typename Vec<T>::type V8;
  __shared__ __attribute__((aligned(16))) T kt[kTile * (DP + 8)], vt[kTile * (DP + 8)];
  int64_t item = work_item(a.work);
  if (item >= a.work) return;
  const int split = SPLIT ? (int)(item % a.splits) : 0;
  if (SPLIT) item /= a.splits;
  const int ct = (int)(item % a.col_tiles);
  const int64_t be = item / a.col_tiles;
  const int b = (int)(be / a.E), e = (int)(be - (int64_t)b * a.E);
  const int lane = threadIdx.x & 63, hi = lane >> 5, wave = threadIdx.x >> 6;
  const int64_t row = (int64_t)ct * (32 * kWaves) + wave * 32 + (lane & 31);
  const bool live = row < a.rows;
  const int g = live ? (int)(row / a.Lq) : 0, i = live ? (int)(row - (int64_t)g * a.Lq) : 0, h = e * a.G + g;
  V8 q[DP / 16];
  load_frags<T, DP>(live ? (const T *)a.q + b * a.qs[0] + i * a.qs[1] + h * a.qs[2] : nullptr, a.D, q);
  const T *kb = (const T *)a.k + b * a.ks[0] + e * a.ks[2], *vb = (const T *)a.v + b * a.vs[0] + e * a.vs[2];
  f32x16 o[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) o[d] = 0.0f;
  float top = -INFINITY, sum = 0.0f;   // of this lane's column; the sum over the rows this lane holds
  Stage<T, DP> ks, vs;
  const int first = SPLIT ? split * a.split_tiles : 0, last = SPLIT && first + a.split_tiles < a.tiles ? first + a.split_tiles : a.tiles;
  walk_tiles(
      a, b, first, last,
      [&](int tile, unsigned long long m) {
        const int64_t at = (int64_t)tile * kTile;
        ks.load(a.D, [&](int r) { return m >> r & 1 ? kb + (at + r) * a.ks[1] : nullptr; });
        vs.load(a.D, [&](int r) { return m >> r & 1 ? vb + (at + r) * a.vs[1] : nullptr; });
      },
      [&]() { ks.store(kt), vs.store(vt); },
      [&](int, unsigned long long m) {
        m = uniform(m);
        f32x16 s[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          s[t] = 0.0f;
#pragma unroll
          for (int d = 0; d < DP / 16; ++d) s[t] = mfma(row_frag<T, DP>(kt, t, d), q[d], s[t]);
        }
        if (m != ~0ull) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const unsigned bits = (unsigned)(m >> (32 * t)) >> (4 * hi);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[t][r] = bits >> (8 * (r / 4) + r % 4) & 1 ? s[t][r] : -INFINITY;
          }
        }
        float mx = s[0][0];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[t][r]);
        mx = fmaxf(mx, other_half(mx));
        const float now = fmaxf(top, mx * a.c);
        if (__any(now > top)) {
          const float f = __builtin_amdgcn_exp2f(top - (now == -INFINITY ? 0.0f : now));
          sum *= f;
#pragma unroll
          for (int d = 0; d < DP / 32; ++d) o[d] *= f;
          top = now;
        }
        const float off = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            s[t][r] = __builtin_amdgcn_exp2f(fmaf(s[t][r], a.c, -off));
            sum += s[t][r];
          }
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const V8 p = to_frag<T>(s[t], half);
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) o[d] = mfma(col_frag<T, DP>(vt, 2 * t + half, d), p, o[d]);
          }
        }
      });
  sum += other_half(sum);
  if (!live) return;
  const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;   // (a NaN stays one)
  if constexpr (SPLIT) {
    const int64_t line = (split * (int64_t)a.B * a.E + be) * a.rows + row;
    float *p = a.part + line * a.D;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at = 32 * d + 8 * r + 4 * hi;
        const float x[4] = {o[d][4 * r] * inv, o[d][4 * r + 1] * inv, o[d][4 * r + 2] * inv, o[d][4 * r + 3] * inv};
        store_n<4>(p + at, a.D - at, x);
      }
    if (hi == 0) a.part_lse[line] = sum == 0.0f ? -INFINITY : top + __builtin_amdgcn_logf(sum);
  } else {
    T *p = (T *)a.out + (((int64_t)b * a.Lq + i) * a.H + h) * a.D;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at = 32 * d + 8 * r + 4 * hi;
        const float x[4] = {o[d][4 * r] * inv, o[d][4 * r + 1] * inv, o[d][4 * r + 2] * inv, o[d][4 * r + 3] * inv};
        store_n<4>(p + at, a.D - at, x);
      }
    if (a.lse && hi == 0) a.lse[be * a.rows + row] = sum == 0.0f ? INFINITY : top + __builtin_amdgcn_logf(sum);
  }
}

// one wave per row: the splits' rows weighted by their share of the sum
template <typename T>
__global__ __launch_bounds__(kBlock) void k_attend_join(AttArgs a) {
  const int64_t lines = (int64_t)a.B * a.E * a.rows, line = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (line >= lines) return;
  const int lane = threadIdx.x & 63;
  float top = -INFINITY;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, a.part_lse[s * lines + line]);
  const float off = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f, x[2] = {0.0f, 0.0f};
  for (int s = 0; s < a.splits; ++s) {
    const float w = __builtin_amdgcn_exp2f(a.part_lse[s * lines + line] - off);
    sum += w;
    for (int k = 0; k < 2; ++k)
      if (lane + 64 * k < a.D) x[k] += w * a.part[(s * lines + line) * a.D + lane + 64 * k];
  }
  const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
  const int64_t be = line / a.rows, row = line - be * a.rows, b = be / a.E, e = be - b * a.E, g = row / a.Lq, i = row - g * a.Lq;
  T *p = (T *)a.out + ((b * a.Lq + i) * a.H + e * a.G + g) * a.D;
  for (int k = 0; k < 2; ++k)
    if (lane + 64 * k < a.D) p[lane + 64 * k] = (T)(x[k] * inv);
  if (a.lse && lane == 0) a.lse[line] = sum == 0.0f ? INFINITY : off + __builtin_amdgcn_logf(sum);
}

// ---- dQ (and delta) ----------------------------------------------------------------------------------------------

template <typename T, int DP, bool SPLIT>
__global__ __launch_bounds__(kBlock, 2) void k_attend_dq(AttArgs a) {
  typedef typename Vec<T>::type V8;
  __shared__ __attribute__((aligned(16))) T kt[kTile * (DP + 8)], vt[kTile * (DP + 8)];
  int64_t item = work_item(a.work);
  if (item >= a.work) return;
  const int split = SPLIT ? (int)(item % a.splits) : 0;
  if (SPLIT) item /= a.splits;
  const int ct = (int)(item % a.col_tiles);
  const int64_t be = item / a.col_tiles;
  const int b = (int)(be / a.E), e = (int)(be - (int64_t)b * a.E);
  const int lane = threadIdx.x & 63, hi = lane >> 5, wave = threadIdx.x >> 6;
  const int64_t row = (int64_t)ct * (32 * kWaves) + wave * 32 + (lane & 31);
  const bool live = row < a.rows;
  const int g = live ? (int)(row / a.Lq) : 0, i = live ? (int)(row - (int64_t)g * a.Lq) : 0, h = e * a.G + g;
  V8 q[DP / 16], go[DP / 16];
  load_frags<T, DP>(live ? (const T *)a.q + b * a.qs[0] + i * a.qs[1] + h * a.qs[2] : nullptr, a.D, q);
  load_frags<T, DP>(live ? (const T *)a.go + b * a.gs[0] + i * a.gs[1] + h * a.gs[2] : nullptr, a.D, go);
  float delta = 0.0f;
  {
    const T *p = live ? (const T *)a.o + (((int64_t)b * a.Lq + i) * a.H + h) * a.D : nullptr;
    V8 o[DP / 16];
    load_frags<T, DP>(p, a.D, o);
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
#pragma unroll
      for (int k = 0; k < 8; ++k) delta += (float)o[s][k] * (float)go[s][k];
    delta += other_half(delta);
  }
  const float lse = live ? a.lse[be * a.rows + row] : INFINITY;
  if (live && hi == 0 && split == 0) a.delta[be * a.rows + row] = delta;
  const T *kb = (const T *)a.k + b * a.ks[0] + e * a.ks[2], *vb = (const T *)a.v + b * a.vs[0] + e * a.vs[2];
  f32x16 dq[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) dq[d] = 0.0f;
  Stage<T, DP> ks, vs;
  const int first = SPLIT ? split * a.split_tiles : 0, last = SPLIT && first + a.split_tiles < a.tiles ? first + a.split_tiles : a.tiles;
  walk_tiles(
      a, b, first, last,
      [&](int tile, unsigned long long m) {
        const int64_t at = (int64_t)tile * kTile;
        ks.load(a.D, [&](int r) { return m >> r & 1 ? kb + (at + r) * a.ks[1] : nullptr; });
        vs.load(a.D, [&](int r) { return m >> r & 1 ? vb + (at + r) * a.vs[1] : nullptr; });
      },
      [&]() { ks.store(kt), vs.store(vt); },
      [&](int, unsigned long long m) {
        m = uniform(m);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          f32x16 s = 0.0f, dp = 0.0f;
#pragma unroll
          for (int d = 0; d < DP / 16; ++d) s = mfma(row_frag<T, DP>(kt, t, d), q[d], s);
#pragma unroll
          for (int d = 0; d < DP / 16; ++d) dp = mfma(row_frag<T, DP>(vt, t, d), go[d], dp);
          const unsigned bits = (unsigned)(m >> (32 * t)) >> (4 * hi);
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            float p = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -lse));
            if (m != ~0ull) p = bits >> (8 * (r / 4) + r % 4) & 1 ? p : 0.0f;
            s[r] = p * (dp[r] - delta);
          }
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const V8 ds = to_frag<T>(s, half);
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) dq[d] = mfma(col_frag<T, DP>(kt, 2 * t + half, d), ds, dq[d]);
          }
        }
      });
  if (!live) return;
  if constexpr (SPLIT) {
    float *p = a.part + ((split * (int64_t)a.B * a.E + be) * a.rows + row) * a.D;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at = 32 * d + 8 * r + 4 * hi;
        const float x[4] = {dq[d][4 * r], dq[d][4 * r + 1], dq[d][4 * r + 2], dq[d][4 * r + 3]};
        store_n<4>(p + at, a.D - at, x);
      }
  } else {
    T *p = (T *)a.dq + (((int64_t)b * a.Lq + i) * a.H + h) * a.D;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at = 32 * d + 8 * r + 4 * hi;
        const float x[4] = {dq[d][4 * r] * a.scale, dq[d][4 * r + 1] * a.scale, dq[d][4 * r + 2] * a.scale, dq[d][4 * r + 3] * a.scale};
        store_n<4>(p + at, a.D - at, x);
      }
  }
}

template <typename T>
__global__ __launch_bounds__(kBlock) void k_attend_dq_join(AttArgs a) {
  const int64_t lines = (int64_t)a.B * a.E * a.rows, line = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (line >= lines) return;
  const int lane = threadIdx.x & 63;
  const int64_t be = line / a.rows, row = line - be * a.rows, b = be / a.E, e = be - b * a.E, g = row / a.Lq, i = row - g * a.Lq;
  T *p = (T *)a.dq + ((b * a.Lq + i) * a.H + e * a.G + g) * a.D;
  for (int k = 0; k < 2; ++k)
    if (lane + 64 * k < a.D) {
      float x = 0.0f;
      for (int s = 0; s < a.splits; ++s) x += a.part[(s * lines + line) * a.D + lane + 64 * k];
      p[lane + 64 * k] = (T)(x * a.scale);
    }
}

// ---- dK, dV ------------------------------------------------------------------------------------------------------

template <typename T, int DP>
__global__ __launch_bounds__(kBlock, DP <= 64 ? 2 : 1) void k_attend_dkv(AttArgs a) {
  typedef typename Vec<T>::type V8;
  __shared__ __attribute__((aligned(16))) T qt[kTile * (DP + 8)], gt[kTile * (DP + 8)];
  __shared__ __attribute__((aligned(16))) float lses[kTile], deltas[kTile];
  const int64_t item = work_item(a.work);
  if (item >= a.work) return;
  const int ct = (int)(item % a.col_tiles);
  const int64_t be = item / a.col_tiles;
  const int b = (int)(be / a.E), e = (int)(be - (int64_t)b * a.E);
  const int lane = threadIdx.x & 63, hi = lane >> 5, wave = threadIdx.x >> 6;
  const int key = ct * (32 * kWaves) + wave * 32 + (lane & 31);
  const bool there = key < a.Lk, on = there && (!a.keep || a.keep[(int64_t)b * a.groups + key / a.per] != 0);
  V8 k[DP / 16], v[DP / 16];
  load_frags<T, DP>(on ? (const T *)a.k + b * a.ks[0] + (int64_t)key * a.ks[1] + e * a.ks[2] : nullptr, a.D, k);
  load_frags<T, DP>(on ? (const T *)a.v + b * a.vs[0] + (int64_t)key * a.vs[1] + e * a.vs[2] : nullptr, a.D, v);
  const bool all = __all(on);
  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) dk[d] = 0.0f, dv[d] = 0.0f;
  const T *qb = (const T *)a.q + b * a.qs[0] + (int64_t)e * a.G * a.qs[2], *gb = (const T *)a.go + b * a.gs[0] + (int64_t)e * a.G * a.gs[2];
  Stage<T, DP> qs, gs;
  float lse = 0.0f, delta = 0.0f;
  const int tiles = __syncthreads_or(on) ? (a.rows + kTile - 1) / kTile : 0;   // (no kept key here: zeros)
  const auto load = [&](int tile) {
    const int at = tile * kTile;
    qs.load(a.D, [&](int r) -> const T * {
      const int row = at + r, g = row / a.Lq;
      return row < a.rows ? qb + (int64_t)(row - g * a.Lq) * a.qs[1] + g * a.qs[2] : nullptr;
    });
    gs.load(a.D, [&](int r) -> const T * {
      const int row = at + r, g = row / a.Lq;
      return row < a.rows ? gb + (int64_t)(row - g * a.Lq) * a.gs[1] + g * a.gs[2] : nullptr;
    });
    if (threadIdx.x < kTile) {
      const int row = at + threadIdx.x;
      lse = row < a.rows ? a.lse[be * a.rows + row] : INFINITY;
      delta = row < a.rows ? a.delta[be * a.rows + row] : 0.0f;
    }
  };
  if (tiles) load(0);
  for (int tile = 0; tile < tiles; ++tile) {
    lds_barrier();
    qs.store(qt), gs.store(gt);
    if (threadIdx.x < kTile) lses[threadIdx.x] = lse, deltas[threadIdx.x] = delta;
    lds_barrier();
    if (tile + 1 < tiles) load(tile + 1);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x16 s = 0.0f, dp = 0.0f;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) s = mfma(row_frag<T, DP>(qt, t, d), k[d], s);
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) dp = mfma(row_frag<T, DP>(gt, t, d), v[d], dp);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int at = 32 * t + 8 * (r / 4) + 4 * hi + r % 4;
        float p = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -lses[at]));
        if (!all) p = on ? p : 0.0f;
        s[r] = p;
        dp[r] = p * (dp[r] - deltas[at]);
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const V8 p = to_frag<T>(s, half), ds = to_frag<T>(dp, half);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
          dv[d] = mfma(col_frag<T, DP>(gt, 2 * t + half, d), p, dv[d]);
          dk[d] = mfma(col_frag<T, DP>(qt, 2 * t + half, d), ds, dk[d]);
        }
      }
    }
  }
  if (!there) return;
  T *pk = (T *)a.dk + (((int64_t)b * a.Lk + key) * a.E + e) * a.D, *pv = (T *)a.dv + (((int64_t)b * a.Lk + key) * a.E + e) * a.D;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int at = 32 * d + 8 * r + 4 * hi;
      const float x[4] = {dk[d][4 * r] * a.scale, dk[d][4 * r + 1] * a.scale, dk[d][4 * r + 2] * a.scale, dk[d][4 * r + 3] * a.scale};
      const float y[4] = {dv[d][4 * r], dv[d][4 * r + 1], dv[d][4 * r + 2], dv[d][4 * r + 3]};
      store_n<4>(pk + at, a.D - at, x);
      store_n<4>(pv + at, a.D - at, y);
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------

int att_args(AttArgs &a, const mvr_attend_params *p) {
  if (!p) return bad("mvr_attend_tokens: params must be given");
  if (p->batch <= 0 || p->queries <= 0 || p->keys <= 0 || p->heads <= 0 || p->kv_heads <= 0 || p->dim <= 0)
    return bad("mvr_attend_tokens: bad shape (every size >= 1)");
  if (p->type != MVR_TYPE_HALF && p->type != MVR_TYPE_BFLOAT) return fail(MVR_ERR_UNSUPPORTED, "mvr_attend_tokens: 16-bit tensors only");
  if (p->dim > 128) return fail(MVR_ERR_UNSUPPORTED, "mvr_attend_tokens: heads of at most 128");
  if (p->heads % p->kv_heads) return bad("mvr_attend_tokens: heads must be a multiple of kv_heads");
  if (p->reserved_) return bad("mvr_attend_tokens: reserved_ must be 0");
  if (p->keep_groups < 0 || (p->keep_groups && p->keys % p->keep_groups)) return bad("mvr_attend_tokens: keep's groups must divide the keys");
  if (!(p->scale > 0.0f) || !(p->scale < INFINITY)) return bad("mvr_attend_tokens: scale must be positive and finite");
  const int64_t rows = (int64_t)(p->heads / p->kv_heads) * p->queries;
  if (rows > 0x7FFFFF00 || p->keys > 0x7FFFFF00) return fail(MVR_ERR_UNSUPPORTED, "mvr_attend_tokens: too many queries or keys");
  a.B = p->batch, a.Lq = p->queries, a.Lk = p->keys, a.H = p->heads, a.E = p->kv_heads, a.G = p->heads / p->kv_heads, a.D = p->dim;
  a.groups = p->keep_groups, a.per = p->keep_groups ? p->keys / p->keep_groups : p->keys;
  a.rows = (int32_t)rows;
  a.scale = p->scale, a.c = p->scale * 1.44269504088896340736f;
  for (int k = 0; k < 3; ++k) a.qs[k] = p->q_stride[k], a.ks[k] = p->k_stride[k], a.vs[k] = p->v_stride[k], a.gs[k] = p->grad_stride[k];
  a.tiles = (p->keys + kTile - 1) / kTile;
  // few columns: the keys are dealt to several workgroups until there are about two per CU, each with four tiles at least
  const int64_t cols = (rows + 32 * kWaves - 1) / (32 * kWaves), blocks = cols * a.B * a.E;
  int64_t splits = 512 / blocks, most = a.tiles / 4;
  splits = splits > most ? most : splits;
  a.splits = splits < 2 ? 1 : (int32_t)splits;
  a.split_tiles = (a.tiles + a.splits - 1) / a.splits;
  a.splits = (a.tiles + a.split_tiles - 1) / a.split_tiles;
  return MVR_OK;
}

size_t lines(const AttArgs &a) { return (size_t)a.B * a.E * a.rows; }
size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }
size_t forward_bytes(const AttArgs &a) { return a.splits > 1 ? align256(lines(a) * a.splits * a.D * 4) + align256(lines(a) * a.splits * 4) : 0; }
size_t backward_bytes(const AttArgs &a) { return align256(lines(a) * 4) + (a.splits > 1 ? align256(lines(a) * a.splits * a.D * 4) : 0); }

// workgroups of 128 columns each, a multiple of 8 for work_item
bool grid_of(AttArgs &a, int64_t columns, int splits, unsigned &blocks) {
  a.col_tiles = (int32_t)((columns + 32 * kWaves - 1) / (32 * kWaves));
  a.work = (int64_t)a.col_tiles * a.B * a.E * splits;
  const int64_t n = (a.work + 7) / 8 * 8;
  blocks = (unsigned)n;
  return n <= 0x7FFFFFFF;
}

template <typename T, int DP>
int launch_forward(AttArgs a, hipStream_t st) {
  unsigned n;
  if (!grid_of(a, a.rows, a.splits, n)) return bad("mvr_attend_tokens_forward: too many workgroups");
  if (a.splits == 1) {
    hipLaunchKernelGGL((k_attend<T, DP, false>), dim3(n), dim3(kBlock), 0, st, a);
    return launched("k_attend");
  }
  hipLaunchKernelGGL((k_attend<T, DP, true>), dim3(n), dim3(kBlock), 0, st, a);
  if (int rc = launched("k_attend")) return rc;
  hipLaunchKernelGGL((k_attend_join<T>), dim3((unsigned)((lines(a) + kWaves - 1) / kWaves)), dim3(kBlock), 0, st, a);
  return launched("k_attend_join");
}

template <typename T, int DP>
int launch_backward(AttArgs a, hipStream_t st) {
  unsigned n;
  if (!grid_of(a, a.rows, a.splits, n)) return bad("mvr_attend_tokens_backward: too many workgroups");
  if (a.splits == 1) {
    hipLaunchKernelGGL((k_attend_dq<T, DP, false>), dim3(n), dim3(kBlock), 0, st, a);
    if (int rc = launched("k_attend_dq")) return rc;
  } else {
    hipLaunchKernelGGL((k_attend_dq<T, DP, true>), dim3(n), dim3(kBlock), 0, st, a);
    if (int rc = launched("k_attend_dq")) return rc;
    hipLaunchKernelGGL((k_attend_dq_join<T>), dim3((unsigned)((lines(a) + kWaves - 1) / kWaves)), dim3(kBlock), 0, st, a);
    if (int rc = launched("k_attend_dq_join")) return rc;
  }
  if (!grid_of(a, a.Lk, 1, n)) return bad("mvr_attend_tokens_backward: too many workgroups");
  hipLaunchKernelGGL((k_attend_dkv<T, DP>), dim3(n), dim3(kBlock), 0, st, a);
  return launched("k_attend_dkv");
}

// heads are padded with zeros to the next of 32, 64, 96, 128
#define MVR_ATT_DIMS(fn, T, a, st) \
  ((a).D <= 32 ? fn<T, 32>(a, st) : (a).D <= 64 ? fn<T, 64>(a, st) : (a).D <= 96 ? fn<T, 96>(a, st) : fn<T, 128>(a, st))

}  // namespace

extern "C" size_t mvr_attend_tokens_workspace_bytes(const mvr_attend_params *params, int32_t backward) {
  AttArgs a = {};
  if (att_args(a, params) != MVR_OK) return 0;
  return backward ? backward_bytes(a) : forward_bytes(a);
}

extern "C" int mvr_attend_tokens_forward(const mvr_attend_params *params, const void *q, const void *k, const void *v, const uint8_t *keep, void *out,
                                         float *lse, void *workspace, size_t workspace_bytes, mvr_stream_t stream) {
  AttArgs a = {};
  if (int rc = att_args(a, params)) return rc;
  if (!q || !k || !v || !out) return bad("mvr_attend_tokens_forward: q, k, v and out must be given");
  if (out == q || out == k || out == v) return bad("mvr_attend_tokens_forward: out must not be an input");
  if ((keep != nullptr) != (params->keep_groups > 0)) return bad("mvr_attend_tokens_forward: keep goes with its groups");
  const size_t need = forward_bytes(a);
  if (need && (!workspace || workspace_bytes < need))
    return fail(MVR_ERR_WORKSPACE, "mvr_attend_tokens_forward: the workspace is smaller than mvr_attend_tokens_workspace_bytes says");
  a.q = q, a.k = k, a.v = v, a.keep = keep, a.out = out, a.lse = lse;
  a.part = (float *)workspace, a.part_lse = (float *)((char *)workspace + align256(lines(a) * a.splits * a.D * 4));
  const hipStream_t st = (hipStream_t)stream;
  return params->type == MVR_TYPE_HALF ? MVR_ATT_DIMS(launch_forward, f16, a, st) : MVR_ATT_DIMS(launch_forward, bf16, a, st);
}

extern "C" int mvr_attend_tokens_backward(const mvr_attend_params *params, const void *q, const void *k, const void *v, const uint8_t *keep,
                                          const void *out, const float *lse, const void *grad_out, void *grad_q, void *grad_k, void *grad_v,
                                          void *workspace, size_t workspace_bytes, mvr_stream_t stream) {
  AttArgs a = {};
  if (int rc = att_args(a, params)) return rc;
  if (!q || !k || !v || !out || !lse || !grad_out || !grad_q || !grad_k || !grad_v)
    return bad("mvr_attend_tokens_backward: every tensor but keep must be given");
  if ((keep != nullptr) != (params->keep_groups > 0)) return bad("mvr_attend_tokens_backward: keep goes with its groups");
  if (!workspace || workspace_bytes < backward_bytes(a))
    return fail(MVR_ERR_WORKSPACE, "mvr_attend_tokens_backward: the workspace is smaller than mvr_attend_tokens_workspace_bytes says");
  a.q = q, a.k = k, a.v = v, a.keep = keep, a.o = out, a.lse = const_cast<float *>(lse), a.go = grad_out, a.dq = grad_q, a.dk = grad_k, a.dv = grad_v;
  a.delta = (float *)workspace, a.part = (float *)((char *)workspace + align256(lines(a) * 4));
  const hipStream_t st = (hipStream_t)stream;
  return params->type == MVR_TYPE_HALF ? MVR_ATT_DIMS(launch_backward, f16, a, st) : MVR_ATT_DIMS(launch_backward, bf16, a, st);
}
