// The tokens of rendered views, where a network takes them up after the renderer and the regulariser: rotary positions with several axes, and the
// norms around a block with its gate and residual scale.  (Attention over the tokens: mvr_attend.hip.)
//
// Both operators are bound by HBM: every kernel here reads each input once and writes each output once, all arithmetic in 32 bits
// (angles in 64, to the fraction of a turn), one rounding at the store.
#include <math.h>

#include "mvr_token_types.h"

using namespace mvr_tok;

namespace {

// ======================================================================================
// rotary positions
// ======================================================================================
//
// Pair i of a head turns by th_i = 2 pi pos[axis(i)] turns_i:  y1 = x1 cos - x2 sin,  y2 = x1 sin + x2 cos.
// The product pos * turns is formed and reduced to a fraction of a turn in 64 bits: at position 1e5 a 32-bit product is off by 4e-3 turns.  The fraction, 1/2 at
// most, is then rounded to 32 bits for sincospi: 2^-26 turns, an angle off by 1.6 2^-24, as much as the functions themselves (float32 results: 1.2 to 1.3 times
// the error of ones with 64-bit sines).
// Backward: dx is dy turned back, and dL/dth_i = x1 dx2 - x2 dx1 (a rotation leaves that determinant alone, so x and dx serve as
// well as y and dy), summed over the heads and, times 2 pi turns_i, over the pairs of an axis — in a fixed order, without atomics.
//
// A workgroup takes `tb` tokens: their cosines and sines go to LDS once (one 64-bit reduction and one sincospi per pair, shared by the
// heads), then thread (token, unit of 16 bytes, head slice) keeps the cosines of its pairs in registers and walks its heads: one
// 16-byte load and store per half of a pair, nothing else in the loop.

constexpr int kBlock = 256;
constexpr int kMaxPairs = 128;

struct RotArgs {
  const void *x, *g;      // x (forward; backward only where the positions' gradient is asked for), grad_out
  void *out;              // out / grad_x, contiguous
  const float *pos;
  float *gpos;            // (B, L, axes) or null
  int64_t xs[3], gs[3], ps[2];
  int64_t rows;           // B * L
  int32_t L, H, D, n;     // n: pairs
  int32_t units, rest;    // 16-byte units of rotated pairs / all units of a head
  int32_t tb, hs;         // tokens and head slices of a workgroup
  int32_t axes, end[4];   // end[a]: first pair behind axis a
  double turns[kMaxPairs];
};

template <typename T, bool INTER, bool BWD, bool GPOS>
__global__ __launch_bounds__(kBlock) void k_rotate_tokens(RotArgs a) {
  constexpr int VE = 16 / sizeof(T);            // elements of a unit's vector
  constexpr int NP = INTER ? VE / 2 : VE;       // pairs of a unit
  constexpr int AHEAD = GPOS ? 2 : 4;           // heads whose loads are in flight
  extern __shared__ float2 cs[];                // [tb][n]; then, with GPOS, the slopes [hs][tb][n] as floats
  const int tid = threadIdx.x;
  const unsigned row0 = blockIdx.x * (unsigned)a.tb, rows = (unsigned)a.rows, L = (unsigned)a.L;
  const int here = (int)(rows - row0 < (unsigned)a.tb ? rows - row0 : (unsigned)a.tb);
  float *slopes = reinterpret_cast<float *>(cs + a.tb * a.n);
  const int u = tid % a.rest, q = tid / a.rest, slice = q % a.hs, t = q / a.hs;
  const bool live = t < here, turned = live && u < a.units;
  const unsigned row = row0 + (live ? t : 0), b = row / L, l = row - b * L;
  const T *in = (const T *)(BWD ? a.g : a.x) + (BWD ? b * a.gs[0] + l * a.gs[1] : b * a.xs[0] + l * a.xs[1]);
  const int64_t in_h = BWD ? a.gs[2] : a.xs[2];
  const T *x = GPOS ? (const T *)a.x + b * a.xs[0] + l * a.xs[1] : nullptr;
  T *out = (T *)a.out + (int64_t)row * a.H * a.D;
  const int i0 = u * NP;                        // first pair
  // where the unit's vectors lie in a head, and how much of them is there
  const int at1 = INTER ? 2 * i0 : i0, at2 = a.n + i0;
  const int left = INTER ? a.D - at1 : a.n - i0;
  const int pairs = a.n - i0;                   // pairs behind it (interleaved: the head's tail in this vector) stay as they are
  Raw<T, VE> v1[AHEAD], v2[AHEAD], x1[AHEAD], x2[AHEAD];
  const auto fetch = [&](int j, int h) {
    v1[j].load(in + h * in_h + at1, left);
    if constexpr (!INTER) v2[j].load(in + h * in_h + at2, left);
    if constexpr (GPOS) {
      x1[j].load(x + h * a.xs[2] + at1, left);
      if constexpr (!INTER) x2[j].load(x + h * a.xs[2] + at2, left);
    }
  };
  if (turned) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (slice + j * a.hs < a.H) fetch(j, slice + j * a.hs);
  }
  // the angles, while the first heads are on their way
  for (int e = tid; e < here * a.n; e += kBlock) {
    const int t1 = e / a.n, i = e - t1 * a.n;
    int axis = 0;
    for (int k = 0; k + 1 < a.axes; ++k) axis += i >= a.end[k];
    const unsigned r1 = row0 + t1, b1 = r1 / L, l1 = r1 - b1 * L;
    const double p = (double)a.pos[b1 * a.ps[0] + l1 * a.ps[1] + axis] * a.turns[i];
    const float r = (float)(p - rint(p));
    float s, c;
    sincospif(2.0f * r, &s, &c);
    cs[e] = make_float2(c, BWD ? -s : s);
  }
  lds_barrier();
  if (turned) {
    float c[NP], s[NP], th[NP];
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const float2 v = k < pairs ? cs[t * a.n + i0 + k] : make_float2(1.0f, 0.0f);
      c[k] = v.x, s[k] = v.y, th[k] = 0.0f;
    }
    for (int h0 = slice; h0 < a.H; h0 += a.hs * AHEAD) {
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int h = h0 + j * a.hs, next = h + a.hs * AHEAD;
        if (h >= a.H) break;
        float v[VE], w[VE], xv[VE], xw[VE];
        v1[j].get(v);
        if constexpr (!INTER) v2[j].get(w);
        if constexpr (GPOS) {
          x1[j].get(xv);
          if constexpr (!INTER) x2[j].get(xw);
        }
        if (next < a.H) fetch(j, next);
#pragma unroll
        for (int k = 0; k < NP; ++k) {
          const float e1 = INTER ? v[2 * k] : v[k], e2 = INTER ? v[2 * k + 1] : w[k];
          const float r1 = e1 * c[k] - e2 * s[k], r2 = e1 * s[k] + e2 * c[k];
          if constexpr (GPOS) {
            const float p1 = INTER ? xv[2 * k] : xv[k], p2 = INTER ? xv[2 * k + 1] : xw[k];
            th[k] += k < pairs ? p1 * r2 - p2 * r1 : 0.0f;
          }
          if constexpr (INTER) {
            v[2 * k] = k < pairs ? r1 : e1;
            v[2 * k + 1] = k < pairs ? r2 : e2;
          } else {
            v[k] = r1, w[k] = r2;
          }
        }
        store_n<VE>(out + (int64_t)h * a.D + at1, left, v);
        if constexpr (!INTER) store_n<VE>(out + (int64_t)h * a.D + at2, left, w);
      }
    }
    if constexpr (GPOS) {
#pragma unroll
      for (int k = 0; k < NP; ++k)
        if (k < pairs) slopes[(slice * a.tb + t) * a.n + i0 + k] = th[k];
    }
  } else if (live) {                            // the head's part behind the pairs
    const int at = (INTER ? a.units * VE : 2 * a.n) + (u - a.units) * VE;
    for (int h = slice; h < a.H; h += a.hs) {
      float v[VE];
      load_n<VE>(in + h * in_h + at, a.D - at, v);
      store_n<VE>(out + (int64_t)h * a.D + at, a.D - at, v);
    }
  }
  if constexpr (GPOS) {
    lds_barrier();
    for (int e = tid; e < here * a.axes; e += kBlock) {
      const int t1 = e / a.axes, ax = e - t1 * a.axes;
      float sum = 0.0f;
      for (int i = ax ? a.end[ax - 1] : 0; i < a.end[ax]; ++i) {
        float th = 0.0f;
        for (int k = 0; k < a.hs; ++k) th += slopes[(k * a.tb + t1) * a.n + i];
        sum += th * (float)(2.0 * M_PI * a.turns[i]);
      }
      a.gpos[(int64_t)(row0 + t1) * a.axes + ax] = sum;
    }
  }
}

int type_size(int t) { return t == MVR_TYPE_FLOAT ? 4 : t == MVR_TYPE_HALF || t == MVR_TYPE_BFLOAT ? 2 : 0; }

int rotary_args(RotArgs &a, const mvr_rotary_params *p, const double *turns) {
  if (!p || !turns) return bad("mvr_rotate_tokens: params and turns must be given");
  if (p->batch <= 0 || p->tokens <= 0 || p->heads <= 0 || p->dim <= 0 || p->dim > 256 || p->heads > (1 << 20))
    return bad("mvr_rotate_tokens: bad shape (batch, tokens, heads >= 1, 1 <= dim <= 256)");
  if (!type_size(p->type)) return bad("mvr_rotate_tokens: unknown type");
  if (p->reserved_) return bad("mvr_rotate_tokens: reserved_ must be 0");
  if (p->axes < 1 || p->axes > 4) return bad("mvr_rotate_tokens: 1 to 4 axes");
  int n = 0;
  for (int k = 0; k < p->axes; ++k) {
    if (p->sections[k] < 1 || p->sections[k] > kMaxPairs) return bad("mvr_rotate_tokens: a section needs at least one pair");
    n += p->sections[k];
    a.end[k] = n;
  }
  if (2 * n > p->dim) return bad("mvr_rotate_tokens: the sections' pairs do not fit the head dimension");
  if (p->interleaved && p->dim % 2) return bad("mvr_rotate_tokens: interleaved pairs need an even head dimension");
  const int ve = 16 / type_size(p->type), np = p->interleaved ? ve / 2 : ve;
  a.rows = (int64_t)p->batch * p->tokens;
  if (a.rows > 0x7FFFFFFF) return fail(MVR_ERR_UNSUPPORTED, "mvr_rotate_tokens: at most 2^31 - 1 tokens in a batch");
  a.L = p->tokens, a.H = p->heads, a.D = p->dim, a.n = n, a.axes = p->axes;
  for (int k = 0; k < 3; ++k) a.xs[k] = p->x_stride[k], a.gs[k] = p->grad_stride[k];
  a.ps[0] = p->position_stride[0], a.ps[1] = p->position_stride[1];
  if (p->interleaved) {
    a.units = (n + np - 1) / np;
    const int in_units = a.units * ve;   // the last unit's vector also holds the tail that fits behind its pairs
    a.rest = a.units + (p->dim > in_units ? (p->dim - in_units + ve - 1) / ve : 0);
  } else {
    a.units = (n + np - 1) / np;
    a.rest = a.units + (p->dim - 2 * n + ve - 1) / ve;
  }
  // two heads a thread: both are on their way while the angles are formed, and a token's heads lie side by side in a wave's accesses
  // (16 x 2352 x 24 heads x 64 bf16, forward / backward with the positions' gradient, us: one head 64 / 146, two 61 / 88, three 64 / 85,
  // four 67 / 90, eight 72 / 94)
  a.hs = (p->heads + 1) / 2;
  while (a.hs > 1 && a.rest * a.hs > kBlock) --a.hs;
  a.tb = kBlock / (a.rest * a.hs);
  if (a.tb > a.rows) a.tb = (int)a.rows;
  if (a.tb < 1) a.tb = 1;
  for (int k = 0; k < n; ++k) a.turns[k] = turns[k];
  return MVR_OK;
}

template <typename T>
int launch_rotary_t(const RotArgs &a, bool inter, bool bwd, hipStream_t st) {
  const int64_t blocks = (a.rows + a.tb - 1) / a.tb;
  const size_t lds = (size_t)a.tb * a.n * (sizeof(float2) + (a.gpos ? a.hs * sizeof(float) : 0));
  const dim3 g((unsigned)blocks), b(kBlock);
  if (!bwd) {
    if (inter) hipLaunchKernelGGL((k_rotate_tokens<T, true, false, false>), g, b, lds, st, a);
    else hipLaunchKernelGGL((k_rotate_tokens<T, false, false, false>), g, b, lds, st, a);
  } else if (!a.gpos) {
    if (inter) hipLaunchKernelGGL((k_rotate_tokens<T, true, true, false>), g, b, lds, st, a);
    else hipLaunchKernelGGL((k_rotate_tokens<T, false, true, false>), g, b, lds, st, a);
  } else {
    if (inter) hipLaunchKernelGGL((k_rotate_tokens<T, true, true, true>), g, b, lds, st, a);
    else hipLaunchKernelGGL((k_rotate_tokens<T, false, true, true>), g, b, lds, st, a);
  }
  return launched("k_rotate_tokens");
}

int launch_rotary(const RotArgs &a, int type, bool inter, bool bwd, mvr_stream_t stream) {
  const hipStream_t st = (hipStream_t)stream;
  return type == MVR_TYPE_FLOAT ? launch_rotary_t<float>(a, inter, bwd, st)
         : type == MVR_TYPE_HALF ? launch_rotary_t<f16>(a, inter, bwd, st) : launch_rotary_t<bf16>(a, inter, bwd, st);
}

// ======================================================================================
// norms around a block
// ======================================================================================
//
//   n = post N(branch)  (or branch),   y = residual + s g n,   z = N(y) weight + bias
// N divides a row by the root of its mean square (+ eps), after taking its mean off for kind "layer".  A row lives in the registers of one
// wave or of several in a workgroup (norm_plan): one read, both norms' statistics by wave sums, one write.
//
// Backward, with r = 1 / std and hats for normed rows:
//   dyt = dy + r_y (dz w - <dz w> - yhat <dz w yhat>)        (<>: mean over the row; the first mean only for "layer")
//   dresidual = dyt,  dn = s g dyt,  dbranch = r_a (dn post - <dn post> - ahat <dn post ahat>)
// and the column sums dweight = sum dz yhat, dbias = sum dz, dpost = sum dn ahat, dgate = sum s post ahat dyt.  A workgroup sums the columns
// of its rows in registers and leaves one line of partial sums; k_norm_columns adds the lines up in a fixed order.  y is had again from the residual
// and the branch where its stored form has 16 bits: yhat and everything that follows would carry its rounding (1.4 times the error of dweight's
// own store); with 32 bits it is read as stored.  Either way the same number of bytes (16 x 2352 x 768 bf16: 82 us, 79 from the stored y).

struct NormArgs {
  const void *residual, *branch, *weight, *bias, *post, *gate;
  const float *scale;
  void *y, *z;
  float *stats;             // (rows, 4): mean and 1 / std of y, of branch
  // backward: residual = y as stored where it has 32 bits, the residual itself where it has 16; dy / dz either may be null
  const void *dy, *dz;
  void *dresidual, *dbranch;
  float *partial;           // (blocks, 4, D): dweight, dbias, dpost, dgate
  int64_t rows, group_rows, scale_rows, block_rows;
  int32_t D, layer, ptype, blocks_per_group;
  float s, eps;
};

constexpr int kV = 4;   // elements of a lane's vector

__device__ __forceinline__ void load_param(const void *p, int type, int64_t at, int left, float (&v)[kV]) {
  if (type == MVR_TYPE_FLOAT) load_n<kV>((const float *)p + at, left, v);
  else if (type == MVR_TYPE_HALF) load_n<kV>((const f16 *)p + at, left, v);
  else load_n<kV>((const bf16 *)p + at, left, v);
}

// sums over the row of K values at once; with WAVES > 1 through LDS, in wave order (two buffers: one barrier a call)
template <int WAVES, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float *lds, int &turn) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = wave_sum(v[k]);
  if constexpr (WAVES > 1) {
    float *at = lds + turn * WAVES * 2;
    turn ^= 1;
    const int wave = threadIdx.x / 64;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) at[wave * 2 + k] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = 0.0f;
      for (int w = 0; w < WAVES; ++w) v[k] += at[w * 2 + k];
    }
  }
}

// mean (0 for rms) and 1 / std of a row held as v; places behind the row hold zeros and are left out of the second sum
template <int WAVES, int NV>
__device__ __forceinline__ float2 row_stats(const float (&v)[NV][kV], const int (&left)[NV], const NormArgs &a, float *lds, int &turn) {
  float m = 0.0f;
  const float inv = 1.0f / (float)a.D;
  if (a.layer) {
    float s[1] = {0.0f};
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int k = 0; k < kV; ++k) s[0] += v[j][k];
    row_sum<WAVES>(s, lds, turn);
    m = s[0] * inv;
  }
  float q[1] = {0.0f};
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int k = 0; k < kV; ++k) {
      const float d = k < left[j] ? v[j][k] - m : 0.0f;
      q[0] += d * d;
    }
  row_sum<WAVES>(q, lds, turn);
  return make_float2(m, 1.0f / sqrtf(q[0] * inv + a.eps));
}

// this wave's (workgroup's) rows: first, first + step, ...; the next row is on its way while one is worked on
template <typename TR, typename TB, int WAVES, int NV>
__global__ __launch_bounds__(WAVES > 1 ? 64 * WAVES : kBlock) void k_add_norm(NormArgs a) {
  __shared__ float lds[4 * WAVES];
  int turn = 0;
  const int lane = WAVES > 1 ? threadIdx.x : threadIdx.x & 63;
  constexpr int kRows = WAVES > 1 ? 1 : kBlock / 64, kLanes = 64 * WAVES;
  const unsigned rows = (unsigned)a.rows, step = gridDim.x * kRows, scale_rows = (unsigned)a.scale_rows, group_rows = (unsigned)a.group_rows;
  int at[NV], left[NV];
  float w[NV][kV], bi[NV][kV], po[NV][kV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    at[j] = (lane + j * kLanes) * kV;
    left[j] = a.D - at[j] < 0 ? 0 : a.D - at[j];
    load_param(a.weight, a.ptype, at[j], left[j], w[j]);
    if (a.bias) load_param(a.bias, a.ptype, at[j], left[j], bi[j]);
    if (a.post) load_param(a.post, a.ptype, at[j], left[j], po[j]);
  }
  Raw<TR, kV> rr[NV];
  Raw<TB, kV> rb[NV];
  float s = 0.0f;
  bool dropped = false;
  const auto fetch = [&](unsigned row) {
    s = a.scale ? a.scale[row / scale_rows] : a.s;
    dropped = s == 0.0f;   // a dropped view's branch is not read: whatever it holds stays out
    const TR *rp = (const TR *)a.residual + (int64_t)row * a.D;
    const TB *bp = (const TB *)a.branch + (int64_t)row * a.D;
#pragma unroll
    for (int j = 0; j < NV; ++j) rr[j].load(rp + at[j], left[j]), rb[j].load(bp + at[j], dropped ? 0 : left[j]);
  };
  unsigned row = __builtin_amdgcn_readfirstlane(blockIdx.x * kRows + (WAVES > 1 ? 0 : threadIdx.x / 64));
  if (row < rows) fetch(row);
  while (row < rows) {
    float v[NV][kV], n[NV][kV], g[NV][kV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      rr[j].get(v[j]), rb[j].get(n[j]);
      if (a.gate) load_param(a.gate, a.ptype, (int64_t)(row / group_rows) * a.D + at[j], left[j], g[j]);
    }
    const float s0 = s;
    const bool gone = dropped;
    const unsigned next = row + step;
    if (next < rows) fetch(next);
    float2 sa = make_float2(0.0f, 1.0f);
    if (a.post) sa = row_stats<WAVES, NV>(n, left, a, lds, turn);
    if (!gone) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < kV; ++k) {
          float t = a.post ? (n[j][k] - sa.x) * sa.y * po[j][k] : n[j][k];
          if (a.gate) t *= g[j][k];
          if (k < left[j]) v[j][k] += s0 * t;
        }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) store_n<kV>((TR *)a.y + (int64_t)row * a.D + at[j], left[j], v[j]);
    const float2 sy = row_stats<WAVES, NV>(v, left, a, lds, turn);
    if (a.stats && lane == 0) *reinterpret_cast<float4 *>(a.stats + (int64_t)row * 4) = make_float4(sy.x, sy.y, sa.x, sa.y);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int k = 0; k < kV; ++k) {
        v[j][k] = (v[j][k] - sy.x) * sy.y * w[j][k];
        if (a.bias) v[j][k] += bi[j][k];
      }
      store_n<kV>((TB *)a.z + (int64_t)row * a.D + at[j], left[j], v[j]);
    }
    row = next;
  }
}

template <typename TR, typename TB, int WAVES, int NV>
__global__ __launch_bounds__(WAVES > 1 ? 64 * WAVES : kBlock) void k_add_norm_backward(NormArgs a) {
  constexpr int kRows = WAVES > 1 ? 1 : kBlock / 64, kLanes = 64 * WAVES;
  __shared__ float lds[4 * WAVES];
  __shared__ float cols[WAVES > 1 ? 1 : kRows][WAVES > 1 ? 1 : kLanes * kV];
  __shared__ float4 params[NV * kLanes][3];   // weight, post_weight, gate: in LDS, the registers go to rows and column sums
  int turn = 0;
  const int lane = WAVES > 1 ? threadIdx.x : threadIdx.x & 63, wave = WAVES > 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const unsigned group = blockIdx.x / (unsigned)a.blocks_per_group, part = blockIdx.x - group * (unsigned)a.blocks_per_group;
  const unsigned scale_rows = (unsigned)a.scale_rows, end_g = (group + 1) * (unsigned)a.group_rows;
  const unsigned first = group * (unsigned)a.group_rows + part * (unsigned)a.block_rows;
  const unsigned last = end_g - first < (unsigned)a.block_rows ? end_g : first + (unsigned)a.block_rows;
  const float inv = 1.0f / (float)a.D;
  int at[NV], left[NV];
  float dw[NV][kV], db[NV][kV], dp[NV][kV], dg[NV][kV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    at[j] = (lane + j * kLanes) * kV;
    left[j] = a.D - at[j] < 0 ? 0 : a.D - at[j];
    float w[kV], po[kV], ga[kV];
    load_param(a.weight, a.ptype, at[j], left[j], w);
    if (a.post) load_param(a.post, a.ptype, at[j], left[j], po);
    if (a.gate) load_param(a.gate, a.ptype, (int64_t)group * a.D + at[j], left[j], ga);
#pragma unroll
    for (int k = 0; k < kV; ++k) {
      if (!a.post) po[k] = 1.0f;
      if (!a.gate) ga[k] = 1.0f;
      dw[j][k] = db[j][k] = dp[j][k] = dg[j][k] = 0.0f;
    }
    // (all waves of a workgroup with rows of their own write the same values)
    float4 *to = params[j * kLanes + lane];
    to[0] = make_float4(w[0], w[1], w[2], w[3]), to[1] = make_float4(po[0], po[1], po[2], po[3]), to[2] = make_float4(ga[0], ga[1], ga[2], ga[3]);
  }
  lds_barrier();
  Raw<TR, kV> ry[NV], rdy[NV];
  Raw<TB, kV> rb[NV], rdz[NV];
  float s = 0.0f;
  bool dropped = false;
  float4 stats;
  const auto fetch = [&](unsigned row) {
    s = a.scale ? a.scale[row / scale_rows] : a.s;
    dropped = s == 0.0f;
    stats = *reinterpret_cast<const float4 *>(a.stats + (int64_t)row * 4);
    const int64_t base = (int64_t)row * a.D;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      ry[j].load((const TR *)a.residual + base + at[j], left[j]);
      rdz[j].load((const TB *)a.dz + base + at[j], a.dz ? left[j] : 0);
      rdy[j].load((const TR *)a.dy + base + at[j], a.dy ? left[j] : 0);
      rb[j].load((const TB *)a.branch + base + at[j], dropped ? 0 : left[j]);
    }
  };
  unsigned row = first + wave;
  if (row < last) fetch(row);
  while (row < last) {
    asm volatile("" ::: "memory");   // (the parameters stay in LDS: hoisted out of the loop they cost a third of the registers)
    float y[NV][kV], n[NV][kV], g[NV][kV], t[NV][kV];
#pragma unroll
    for (int j = 0; j < NV; ++j) ry[j].get(y[j]), rb[j].get(n[j]), rdz[j].get(g[j]), rdy[j].get(t[j]);
    const float s0 = s;
    const bool gone = dropped;
    const float4 st = stats;
    const unsigned next = row + kRows;
    if (next < last) fetch(next);
    float m[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const float4 w4 = params[j * kLanes + lane][0];
      const float w[kV] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
      for (int k = 0; k < kV; ++k) n[j][k] = gone || k >= left[j] ? 0.0f : a.post ? (n[j][k] - st.z) * st.w : n[j][k];   // ahat (or the branch)
      if constexpr (sizeof(TR) == 2) {   // y from the residual
        const float4 p4 = params[j * kLanes + lane][1], g4 = params[j * kLanes + lane][2];
        const float po[kV] = {p4.x, p4.y, p4.z, p4.w}, ga[kV] = {g4.x, g4.y, g4.z, g4.w};
#pragma unroll
        for (int k = 0; k < kV; ++k) y[j][k] += gone ? 0.0f : s0 * (n[j][k] * po[k] * ga[k]);
      }
#pragma unroll
      for (int k = 0; k < kV; ++k) {
        y[j][k] = k < left[j] ? (y[j][k] - st.x) * st.y : 0.0f;   // yhat
        dw[j][k] += g[j][k] * y[j][k];
        db[j][k] += g[j][k];
        g[j][k] *= w[k];
        m[0] += g[j][k] * y[j][k];
        m[1] += g[j][k];
      }
    }
    row_sum<WAVES>(m, lds, turn);
    const float m0 = m[0] * inv, m1 = a.layer ? m[1] * inv : 0.0f;
    float d[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const float4 p4 = params[j * kLanes + lane][1], g4 = params[j * kLanes + lane][2];
      const float po[kV] = {p4.x, p4.y, p4.z, p4.w}, ga[kV] = {g4.x, g4.y, g4.z, g4.w};
#pragma unroll
      for (int k = 0; k < kV; ++k) {
        t[j][k] += st.y * (g[j][k] - m1 - y[j][k] * m0);          // dyt
        const float hat = n[j][k];
        const float u = !gone && k < left[j] ? s0 * t[j][k] : 0.0f;   // (0 times an infinite dyt is not 0)
        dg[j][k] += u * po[k] * hat;
        const float dn = u * ga[k];
        dp[j][k] += dn * hat;
        g[j][k] = dn * po[k];
        d[0] += g[j][k] * hat;
        d[1] += g[j][k];
      }
      store_n<kV>((TR *)a.dresidual + (int64_t)row * a.D + at[j], left[j], t[j]);
    }
    if (a.post) {
      row_sum<WAVES>(d, lds, turn);
      const float d0 = d[0] * inv, d1 = a.layer ? d[1] * inv : 0.0f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < kV; ++k) g[j][k] = gone ? 0.0f : st.w * (g[j][k] - d1 - n[j][k] * d0);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) store_n<kV>((TB *)a.dbranch + (int64_t)row * a.D + at[j], left[j], g[j]);
    row = next;
  }
  if (!a.partial) return;
  float *line = a.partial + (int64_t)blockIdx.x * 4 * a.D;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float v[kV];
#pragma unroll
      for (int k = 0; k < kV; ++k) v[k] = q == 0 ? dw[j][k] : q == 1 ? db[j][k] : q == 2 ? dp[j][k] : dg[j][k];
      if constexpr (WAVES > 1) {
        store_n<kV>(line + q * a.D + at[j], left[j], v);
      } else {   // the four waves' rows, in wave order
        lds_barrier();
#pragma unroll
        for (int k = 0; k < kV; ++k) cols[wave][lane * kV + k] = v[k];
        lds_barrier();
        const int e = threadIdx.x, c = j * kLanes * kV + e;
        if (c < a.D) line[q * a.D + c] = (cols[0][e] + cols[1][e]) + (cols[2][e] + cols[3][e]);
      }
    }
  }
}

// 64 columns of one of the four sums: sixteen waves add the lines k, k + 16, ..., then wave 0 adds the waves' sums up
constexpr int kColumns = 64;
__global__ __launch_bounds__(1024) void k_norm_columns(const float *partial, int32_t D, int32_t blocks, int32_t blocks_per_group, int32_t ptype,
                                                       void *dweight, void *dbias, void *dpost, void *dgate) {
  __shared__ float lds[16][kColumns];
  const int q = blockIdx.y < 3 ? blockIdx.y : 3;
  const int64_t group = blockIdx.y < 3 ? 0 : blockIdx.y - 3;
  void *out = q == 0 ? dweight : q == 1 ? dbias : q == 2 ? dpost : dgate;
  if (!out) return;
  const int first = q == 3 ? (int)group * blocks_per_group : 0, last = q == 3 ? first + blocks_per_group : blocks;
  const int wave = threadIdx.x / kColumns, lane = threadIdx.x % kColumns, c = blockIdx.x * kColumns + lane;
  float s = 0.0f;
  if (c < D) {
#pragma unroll 8
    for (int k = first + wave; k < last; k += 16) s += partial[((int64_t)k * 4 + q) * D + c];
  }
  lds[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && c < D) {
    s = 0.0f;
    for (int k = 0; k < 16; ++k) s += lds[k][lane];
    const int64_t at = group * D + c;
    if (ptype == MVR_TYPE_FLOAT) ((float *)out)[at] = s;
    else if (ptype == MVR_TYPE_HALF) ((f16 *)out)[at] = (f16)s;
    else ((bf16 *)out)[at] = (bf16)s;
  }
}

int norm_args(NormArgs &a, const mvr_norm_params *p) {
  if (!p) return bad("mvr_add_norm_tokens: params must be given");
  if (p->rows <= 0 || p->dim <= 0 || p->dim > 8192) return bad("mvr_add_norm_tokens: rows >= 1 and 1 <= dim <= 8192");
  if (p->rows > 0x7FFF0000) return fail(MVR_ERR_UNSUPPORTED, "mvr_add_norm_tokens: too many rows");
  const int r = p->residual_type, b = p->branch_type;
  if (!type_size(r) || !type_size(b) || !type_size(p->param_type)) return bad("mvr_add_norm_tokens: unknown type");
  if (r != b && r != MVR_TYPE_FLOAT) return fail(MVR_ERR_UNSUPPORTED, "mvr_add_norm_tokens: the residual has the branch's type or 32 bits");
  if (p->reserved_) return bad("mvr_add_norm_tokens: reserved_ must be 0");
  if (p->kind != 0 && p->kind != 1) return bad("mvr_add_norm_tokens: kind is 0 (rms) or 1 (layer)");
  if (p->gate_groups < 0 || p->scale_groups < 0 || (p->gate_groups && p->rows % p->gate_groups) || (p->scale_groups && p->rows % p->scale_groups))
    return bad("mvr_add_norm_tokens: the groups of gate and scale must divide the rows");
  if (!(p->eps >= 0.0f)) return bad("mvr_add_norm_tokens: eps must not be negative");
  a.rows = p->rows, a.D = p->dim, a.layer = p->kind, a.ptype = p->param_type, a.s = p->scale, a.eps = p->eps;
  a.group_rows = p->gate_groups ? p->rows / p->gate_groups : p->rows;
  a.scale_rows = p->scale_groups ? p->rows / p->scale_groups : p->rows;
  return MVR_OK;
}

// 256 elements of a row per wave and vector.  Rows of up to 768 lie in one wave's registers (16 x 2352 x 768 bf16, forward / backward: 55.5 / 82 us;
// a row over the three waves of a workgroup 69 / 82 with its columns, where the backward of one wave a row took 79); wider ones take a workgroup:
// 64 x 3920 x 1024 forward 586 us, with one wave a row 622.
// Grids hold as many workgroups as are resident at once (256 CUs by what the registers allow) and every wave runs through its rows: a second,
// partly filled round costs more than it balances (backward at 768, before y was formed again: 512 workgroups 79 us, 768 101, 1024 87).
struct NormPlan { int32_t waves, vectors, forward, backward; };
inline NormPlan norm_plan(int32_t D) {
  return D <= 256 ? NormPlan{1, 1, 2048, 1280} : D <= 512 ? NormPlan{1, 2, 1280, 768} : D <= 768 ? NormPlan{1, 3, 1024, 512}
         : D <= 1024 ? NormPlan{4, 1, 2048, 768} : D <= 2048 ? NormPlan{4, 2, 1280, 768} : D <= 4096 ? NormPlan{8, 2, 512, 256} : NormPlan{8, 4, 256, 256};
}

// the backward's workgroups: each has a run of rows of one gate group
void norm_blocks(const mvr_norm_params *p, int64_t &per_group, int64_t &rows_each, int64_t &blocks) {
  const NormPlan plan = norm_plan(p->dim);
  const int64_t groups = p->gate_groups ? p->gate_groups : 1, rows = p->rows / groups;
  const int64_t least = plan.waves > 1 ? 2 : 8;   // rows of a workgroup: below, the partial sums would weigh more than the rows
  per_group = (plan.backward + groups - 1) / groups;
  if (per_group > (rows + least - 1) / least) per_group = (rows + least - 1) / least;
  rows_each = (rows + per_group - 1) / per_group;
  per_group = (rows + rows_each - 1) / rows_each;
  blocks = per_group * groups;
}

template <typename TR, typename TB>
int launch_norm(const NormArgs &a, hipStream_t st) {
  const NormPlan plan = norm_plan(a.D);
  const int64_t blocks = plan.waves > 1 ? a.rows : (a.rows + 3) / 4;
  const dim3 g((unsigned)(blocks < plan.forward ? blocks : plan.forward)), b(plan.waves > 1 ? 64 * plan.waves : kBlock);
  switch (plan.waves * 10 + plan.vectors) {
    case 11: hipLaunchKernelGGL((k_add_norm<TR, TB, 1, 1>), g, b, 0, st, a); break;
    case 12: hipLaunchKernelGGL((k_add_norm<TR, TB, 1, 2>), g, b, 0, st, a); break;
    case 13: hipLaunchKernelGGL((k_add_norm<TR, TB, 1, 3>), g, b, 0, st, a); break;
    case 41: hipLaunchKernelGGL((k_add_norm<TR, TB, 4, 1>), g, b, 0, st, a); break;
    case 42: hipLaunchKernelGGL((k_add_norm<TR, TB, 4, 2>), g, b, 0, st, a); break;
    case 82: hipLaunchKernelGGL((k_add_norm<TR, TB, 8, 2>), g, b, 0, st, a); break;
    default: hipLaunchKernelGGL((k_add_norm<TR, TB, 8, 4>), g, b, 0, st, a);
  }
  return launched("k_add_norm");
}

template <typename TR, typename TB>
int launch_norm_backward(const NormArgs &a, int64_t blocks, hipStream_t st) {
  const NormPlan plan = norm_plan(a.D);
  const dim3 g((unsigned)blocks), b(plan.waves > 1 ? 64 * plan.waves : kBlock);
  switch (plan.waves * 10 + plan.vectors) {
    case 11: hipLaunchKernelGGL((k_add_norm_backward<TR, TB, 1, 1>), g, b, 0, st, a); break;
    case 12: hipLaunchKernelGGL((k_add_norm_backward<TR, TB, 1, 2>), g, b, 0, st, a); break;
    case 13: hipLaunchKernelGGL((k_add_norm_backward<TR, TB, 1, 3>), g, b, 0, st, a); break;
    case 41: hipLaunchKernelGGL((k_add_norm_backward<TR, TB, 4, 1>), g, b, 0, st, a); break;
    case 42: hipLaunchKernelGGL((k_add_norm_backward<TR, TB, 4, 2>), g, b, 0, st, a); break;
    case 82: hipLaunchKernelGGL((k_add_norm_backward<TR, TB, 8, 2>), g, b, 0, st, a); break;
    default: hipLaunchKernelGGL((k_add_norm_backward<TR, TB, 8, 4>), g, b, 0, st, a);
  }
  return launched("k_add_norm_backward");
}

#define MVR_NORM_TYPES(fn, p, ...)                                                                                                        \
  ((p)->residual_type == MVR_TYPE_FLOAT                                                                                                   \
       ? ((p)->branch_type == MVR_TYPE_FLOAT ? fn<float, float>(__VA_ARGS__)                                                              \
                                             : (p)->branch_type == MVR_TYPE_HALF ? fn<float, f16>(__VA_ARGS__) : fn<float, bf16>(__VA_ARGS__)) \
       : (p)->residual_type == MVR_TYPE_HALF ? fn<f16, f16>(__VA_ARGS__) : fn<bf16, bf16>(__VA_ARGS__))

}  // namespace

extern "C" int mvr_rotate_tokens_forward(const mvr_rotary_params *params, const double *turns, const void *x, const float *positions, void *out,
                                         mvr_stream_t stream) {
  RotArgs a = {};
  if (!x || !positions || !out || x == out) return bad("mvr_rotate_tokens_forward: x, positions and out must be given, x and out distinct");
  if (int rc = rotary_args(a, params, turns)) return rc;
  a.x = x, a.pos = positions, a.out = out;
  return launch_rotary(a, params->type, params->interleaved != 0, false, stream);
}

extern "C" int mvr_rotate_tokens_backward(const mvr_rotary_params *params, const double *turns, const void *x, const float *positions,
                                          const void *grad_out, void *grad_x, float *grad_positions, mvr_stream_t stream) {
  RotArgs a = {};
  if (!positions || !grad_out || !grad_x || grad_out == grad_x) return bad("mvr_rotate_tokens_backward: positions, grad_out and grad_x must be given, the last two distinct");
  if ((x == nullptr) != (grad_positions == nullptr)) return bad("mvr_rotate_tokens_backward: x and grad_positions go together");
  if (int rc = rotary_args(a, params, turns)) return rc;
  a.x = x, a.g = grad_out, a.pos = positions, a.out = grad_x, a.gpos = grad_positions;
  return launch_rotary(a, params->type, params->interleaved != 0, true, stream);
}

extern "C" size_t mvr_add_norm_tokens_workspace_bytes(const mvr_norm_params *params) {
  NormArgs a = {};
  if (norm_args(a, params) != MVR_OK) return 0;
  int64_t per, each, blocks;
  norm_blocks(params, per, each, blocks);
  return (size_t)blocks * 4 * params->dim * sizeof(float);
}

extern "C" int mvr_add_norm_tokens_forward(const mvr_norm_params *params, const void *residual, const void *branch, const void *weight,
                                           const void *bias, const void *post_weight, const void *gate, const float *scale, void *y, void *z,
                                           float *stats, mvr_stream_t stream) {
  NormArgs a = {};
  if (int rc = norm_args(a, params)) return rc;
  if (!residual || !branch || !weight || !y || !z) return bad("mvr_add_norm_tokens_forward: residual, branch, weight, y and z must be given");
  if ((gate != nullptr) != (params->gate_groups > 0) || (scale != nullptr) != (params->scale_groups > 0))
    return bad("mvr_add_norm_tokens_forward: gate and scale go with their groups");
  if (z == y || z == residual || z == branch || y == branch) return bad("mvr_add_norm_tokens_forward: y and z must not overlap each other or the inputs");
  a.residual = residual, a.branch = branch, a.weight = weight, a.bias = bias, a.post = post_weight, a.gate = gate, a.scale = scale;
  a.y = y, a.z = z, a.stats = stats;
  return MVR_NORM_TYPES(launch_norm, params, a, (hipStream_t)stream);
}

extern "C" int mvr_add_norm_tokens_backward(const mvr_norm_params *params, const void *y, const void *branch, const void *weight,
                                            const void *post_weight, const void *gate, const float *scale, const float *stats, const void *grad_y,
                                            const void *grad_z, void *grad_residual, void *grad_branch, void *grad_weight, void *grad_bias,
                                            void *grad_post_weight, void *grad_gate, void *workspace, size_t workspace_bytes,
                                            mvr_stream_t stream) {
  NormArgs a = {};
  if (int rc = norm_args(a, params)) return rc;
  if (!y || !branch || !weight || !stats || (!grad_y && !grad_z) || !grad_residual || !grad_branch)
    return bad("mvr_add_norm_tokens_backward: y_or_residual, branch, weight, stats, one of grad_y and grad_z, grad_residual and grad_branch must be given");
  if ((gate != nullptr) != (params->gate_groups > 0) || (scale != nullptr) != (params->scale_groups > 0))
    return bad("mvr_add_norm_tokens_backward: gate and scale go with their groups");
  if ((grad_gate && !gate) || (grad_post_weight && !post_weight)) return bad("mvr_add_norm_tokens_backward: a gradient of a parameter that is not there");
  int64_t per, each, blocks;
  norm_blocks(params, per, each, blocks);
  if (blocks > 0x7FFFFFFF || params->gate_groups > 65000) return bad("mvr_add_norm_tokens_backward: too many gate groups");
  const bool columns = grad_weight || grad_bias || grad_post_weight || grad_gate;
  if (columns && (!workspace || workspace_bytes < (size_t)blocks * 4 * params->dim * sizeof(float)))
    return fail(MVR_ERR_WORKSPACE, "mvr_add_norm_tokens_backward: the workspace is smaller than mvr_add_norm_tokens_workspace_bytes says");
  a.residual = y, a.branch = branch, a.weight = weight, a.post = post_weight, a.gate = gate, a.scale = scale;
  a.stats = const_cast<float *>(stats), a.dy = grad_y, a.dz = grad_z, a.dresidual = grad_residual, a.dbranch = grad_branch;
  a.partial = columns ? (float *)workspace : nullptr;
  a.blocks_per_group = (int32_t)per, a.block_rows = each;
  if (int rc = MVR_NORM_TYPES(launch_norm_backward, params, a, blocks, (hipStream_t)stream)) return rc;
  if (!columns) return MVR_OK;
  const dim3 g((unsigned)((params->dim + kColumns - 1) / kColumns), 3 + (grad_gate ? (unsigned)params->gate_groups : 0));
  hipLaunchKernelGGL(k_norm_columns, g, dim3(1024), 0, (hipStream_t)stream, a.partial, params->dim, (int32_t)blocks, (int32_t)per,
                     params->param_type, grad_weight, grad_bias, grad_post_weight, grad_gate);
  return launched("k_norm_columns");
}
