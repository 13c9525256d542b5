// Attention over view tokens, forward and backward, for 16-bit tensors:
//   S = scale q k^T over the kept keys,  P = exp(S - lse),  O = P v
//   dV = P^T dO,  dS = P (dO v^T - delta),  delta = rowsum(dO O),  dQ = scale dS k,  dK = scale dS^T q
// One pass over the keys with the running maximum and sum; nothing of size queries x keys is ever stored: the backward recomputes the
// probabilities from q, k and lse.  Sums, maxima and exponentials are 32 bits wide; P and dS are rounded to the tensors' type where they
// enter a matrix instruction: half a step of the type relative to each, as of the inputs, and not where few keys make it count (FINE, at k_attend).
// The forward's P lies in [0, 2^8], as its maximum may lag.  In float16, whose step stops shrinking at 2^-14, P and dS enter times a power of two
// that brings them to the top of its range, and the 32-bit sums are divided by it (at kLift).
//
// All three kernels have one shape.  A wave owns columns — queries (forward: 32 or two times 32, dQ: 32) or keys (dK/dV: 32 or 16) — and walks
// the other side in tiles that its workgroup stages in LDS.  Scores come as tile x columns from v_mfma_f32_32x32x16: a lane then holds 16 scores of ONE column (rows 8 (r / 4) +
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

typedef float f32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

struct AttArgs {
  const void *q, *k, *v, *o, *go;
  const uint8_t *keep;
  void *out, *dq, *dk, *dv;
  void *rest;                    // what out's rounding left, in its type and layout; or null
  float *lse;                    // (B, heads, queries): log2 of the sum of exp2(scale log2(e) q k); +inf for a row without keys
  float *delta;                  // the same shape
  float *part, *part_lse;        // splits over the keys: (splits, B kv_heads rows, D) and (splits, B kv_heads rows); over the rows: (row_splits, 2, B keys kv_heads, D)
  int64_t qs[3], ks[3], vs[3], gs[3];
  int32_t B, Lq, Lk, H, E, G, D;   // E: kv heads, G: heads of a group
  int32_t groups, per;           // keep: (B, groups), `per` keys each
  int32_t rows;                  // G * Lq
  int32_t tiles, splits, split_tiles, col_tiles;
  int32_t row_splits, row_split_tiles;   // of the tiles of rows that dK and dV walk
  int32_t wide;                  // two columns of 32 queries a wave
  int32_t rows_whole;            // whole, and a group's heads of fewer queries than a tile holds do not share tiles
  int32_t whole;                 // D a multiple of 8 and a tile's rows within 32-bit offsets: tiles are loaded in whole chunks
  int64_t work;                  // workgroups with something to do
  float c, scale;                // scale log2(e)
  double per_inverse;            // 1 / per
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

// How a tile lies in LDS: rows of 4, 8 or 16 chunks of 16 bytes, chunk c of row r at c ^ swizzle(r), so that no way of reading it meets a bank
// twice: 16 rows at one chunk (row_frag), 4 rows at 4 chunks or 8 rows at 2 (col_frag) each fall on 16 different bank groups of the 64 banks.
template <int DP>
struct Layout {
  static constexpr int kChunks = DP <= 32 ? 4 : DP <= 64 ? 8 : 16, kPitch = 8 * kChunks, kSize = kTile * kPitch;
  static __device__ __forceinline__ int swizzle(int r) {
    const int low = (r >> 2 & 1) << 1 | (r >> 3 & 1);
    return DP <= 32 ? low : DP <= 64 ? (r >> 1 & 1) << 2 | low : (r & 3) << 2 | low;
  }
};

// A tile of kTile rows on its way from memory to LDS
template <typename T, int DP>
struct Stage {
  static constexpr int kPerRow = DP / 8, kChunks = kTile * kPerRow / kBlock;   // (a whole number for 32, 64, 96 and 128)
  static constexpr bool kEven = kBlock % kPerRow == 0;   // a thread's chunks lie in one column, kBlock / kPerRow rows apart
  u32x4 r[kChunks];
  __device__ __forceinline__ Stage() {
#pragma unroll
    for (int k = 0; k < kChunks; ++k) r[k] = u32x4{0, 0, 0, 0};
  }
  // D a multiple of 8, rows `stride` elements apart, the last of them again for what lies behind it: one way for whole tiles and ends, as loads
  // on two ways into the same registers are copied, and waited for, where the ways meet
  __device__ __forceinline__ void load(const T *base, unsigned stride, int D, unsigned last) {
    if constexpr (kEven) {
      const unsigned i = threadIdx.x / kPerRow, c = threadIdx.x % kPerRow * 8;
      if (c < (unsigned)D) {   // (chunks behind a head stay the zeros they are)
        unsigned at = i * stride + c;
        const unsigned end = last * stride + c;
        asm volatile("" : "+v"(at));   // (one address is kept through the loop, not one per chunk)
#pragma unroll
        for (int k = 0; k < kChunks; ++k) {
          const unsigned x = at + k * (kBlock / kPerRow) * stride;
          __builtin_memcpy(&r[k], base + (x < end ? x : end), 16);
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < kChunks; ++k) {
        const unsigned e = threadIdx.x + k * kBlock, i = e / kPerRow, c = e % kPerRow * 8;
        if (c < (unsigned)D) __builtin_memcpy(&r[k], base + (i < last ? i : last) * stride + c, 16);
      }
    }
  }
  // `row` gives a row's address, or null for a row of zeros
  template <typename Row>
  __device__ __forceinline__ void load_rows(int D, Row row) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));   // (its addresses are not to be kept in registers all through the loop)
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const int e = tid + k * kBlock, i = e / kPerRow, c = e % kPerRow * 8;
      const T *p = row(i);
      r[k] = load16(p + c, p ? D - c : 0);
    }
  }
  // rows whose bit is not set become zeros
  __device__ __forceinline__ void store(T *lds, unsigned long long rows) const {
    const int i0 = threadIdx.x / kPerRow, at0 = i0 * Layout<DP>::kPitch + (threadIdx.x % kPerRow ^ Layout<DP>::swizzle(i0)) * 8;
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const int e = threadIdx.x + k * kBlock, i = e / kPerRow;
      u32x4 x = r[k];
      if (rows != ~0ull && !(rows >> (i & 63) & 1)) x = u32x4{0, 0, 0, 0};
      // (whole multiples of 16 rows apart the swizzle is the same)
      const int at = kEven && kBlock / kPerRow % 16 == 0 ? at0 + k * (kBlock / kPerRow) * Layout<DP>::kPitch
                                                          : i * Layout<DP>::kPitch + (e % kPerRow ^ Layout<DP>::swizzle(i)) * 8;
      *reinterpret_cast<u32x4 *>(lds + at) = x;
    }
  }
};

// Where this lane reads a tile.  A swizzled address is a base with bits flipped, so three bases give all of them; `at` makes fresh copies for one
// step: addresses that follow from them are not kept in registers all through a loop.
typedef __attribute__((address_space(3))) char lds_char;
template <int DP>
struct Reader {
  static constexpr int kRow = 2 * Layout<DP>::kPitch, kBytes = kTile * kRow;   // of 16-bit elements
  unsigned row, col, col8;
  // 32 x 32 x 16: row_frag has the tile's rows 32 t + (lane % 32) as its rows, d = 16 s + 8 (lane / 32) + 0..7 as its depth;
  // col_frag d = 32 db + (lane % 32) as its rows, the tile's rows 16 s + 4 (lane / 32) + {0..3, 8..11} as its depth
  static __device__ __forceinline__ Reader wide(const void *lds) {
    const unsigned lane = threadIdx.x & 63, i = lane & 31, j = 4 * (lane >> 5) + (lane >> 2 & 3), x = (lane >> 4 & 1) * 2 + (lane >> 1 & 1);
    const unsigned base = (unsigned)(size_t)(lds_char *)lds;
    Reader r;
    r.row = base + i * kRow + ((lane >> 5) ^ Layout<DP>::swizzle(i)) * 16;
    r.col = base + j * kRow + (x ^ Layout<DP>::swizzle(j)) * 16 + 8 * (lane & 1);
    r.col8 = base + (j + 8) * kRow + (x ^ Layout<DP>::swizzle(j + 8)) * 16 + 8 * (lane & 1);
    return r;
  }
  // 16 x 16 x 32: rows 16 b + (lane % 16), d = 32 s + 8 (lane / 16) + 0..7;  d = 16 db + (lane % 16), rows 32 t + 4 (lane / 16) + {0..3, 16..19}
  static __device__ __forceinline__ Reader narrow(const void *lds) {
    const unsigned lane = threadIdx.x & 63, i = lane & 15, j = 4 * (lane >> 4) + (lane >> 2 & 3), base = (unsigned)(size_t)(lds_char *)lds;
    Reader r;
    r.row = base + i * kRow + ((lane >> 4) ^ Layout<DP>::swizzle(i)) * 16;
    r.col = base + j * kRow + ((lane >> 1 & 1) ^ Layout<DP>::swizzle(j)) * 16 + 8 * (lane & 1);
    r.col8 = 0;
    return r;
  }
  __device__ __forceinline__ Reader at(int buffer) const {   // of the two tiles of a buffer, the first
    Reader r = {row + buffer * 2 * kBytes, col + buffer * 2 * kBytes, col8 + buffer * 2 * kBytes};
    asm volatile("" : "+v"(r.row), "+v"(r.col), "+v"(r.col8));
    return r;
  }
  template <typename V>
  static __device__ __forceinline__ V load(unsigned at) {
    return *(const __attribute__((address_space(3))) V *)(lds_char *)(size_t)at;
  }
  template <typename V>
  static __device__ __forceinline__ V load_columns(unsigned at, unsigned more) {
    typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
    union { i16x4 h[2]; V v; } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(lds_char *)(size_t)at);
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(lds_char *)(size_t)more);
    return u.v;
  }
};
// the operands of one sub-tile of 32 rows, of a buffer's first or second tile
template <typename T, int DP>
__device__ __forceinline__ void row_frags(const Reader<DP> &r, int which, int t, typename Vec<T>::type (&f)[DP / 16]) {
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) f[s] = Reader<DP>::template load<typename Vec<T>::type>((r.row ^ 32 * s) + which * r.kBytes + 32 * t * r.kRow);
}
template <typename T, int DP>
__device__ __forceinline__ void col_frags(const Reader<DP> &r, int which, int t, typename Vec<T>::type (&f)[2][DP / 32]) {
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) {
      const int off = which * r.kBytes + (32 * t + 16 * half) * r.kRow;
      f[half][d] = Reader<DP>::template load_columns<typename Vec<T>::type>((r.col ^ 64 * d) + off, (r.col8 ^ 64 * d) + off);
    }
}
// Nothing moves across: operands of the next products are not all read at once (the registers are full)
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }

template <typename T>
__device__ __forceinline__ typename Vec<T>::type to_frag(const f32x16 &x, int half) {
  typename Vec<T>::type v;
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = (T)x[8 * half + k];
  return v;
}
// what to_frag's rounding leaves
template <typename T>
__device__ __forceinline__ typename Vec<T>::type rest_frag(const f32x16 &x, int half) {
  typename Vec<T>::type v;
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = (T)(x[8 * half + k] - (float)(T)x[8 * half + k]);
  return v;
}
// x + the sum of an operand's eight values
__device__ __forceinline__ float add_frag(bf16x8 p, float x) {
  typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 one = {(bf16)1.0f, (bf16)1.0f};
  bf16x2 h[4];
  __builtin_memcpy(h, &p, 16);
#pragma unroll
  for (int k = 0; k < 4; ++k) x = __builtin_amdgcn_fdot2_f32_bf16(h[k], one, x, false);
  return x;
}
__device__ __forceinline__ float add_frag(f16x8 p, float x) {
  typedef f16 f16x2 __attribute__((ext_vector_type(2)));
  const f16x2 one = {(f16)1.0f, (f16)1.0f};
  f16x2 h[4];
  __builtin_memcpy(h, &p, 16);
#pragma unroll
  for (int k = 0; k < 4; ++k) x = __builtin_amdgcn_fdot2(h[k], one, x, false);
  return x;
}
// Powers of two for float16.  A row's P over some thousand keys is about 2^-12 and dS = P (dP - delta) smaller still by what a loss' gradient is
// below 1: rounded as they are, most would lie under 2^-14, where float16 keeps 2^-24 of anything (2352 keys, dO of 1e-3: dQ and dK off by 6 and 4 times
// the store's own rounding; times these powers 1.1).
// P: 2^kLift in the forward, where it reaches 2^kSlack without; 2^kLiftP in dK and dV, where it reaches 1.  Both come with the exponent, for nothing.
// dS: one power per column (a query's in dQ, a key's in dK), the largest that keeps |dS| below kMost; like the running maximum it is found on the way:
// it starts at 2^kStart, and where a value leaves the range all of the column so far is multiplied down until the largest is at kAim.  Powers of two: nothing
// else is rounded.  bfloat16 has the exponents of 32 bits and needs none of it.
// Forward and gradients of float16 with and without: 16 x 2352 tokens, 12 heads of 64, 1344 / 1296 us; 8 x 3920, 16 heads of 128, 5192 / 5106.
template <typename T> constexpr bool kNarrow = false;
template <> constexpr bool kNarrow<f16> = true;
template <typename T> constexpr float kLift = kNarrow<T> ? 7.0f : 0.0f;
template <typename T> constexpr float kLiftP = kNarrow<T> ? 14.0f : 0.0f;
constexpr float kStart = 60.0f, kMost = 32768.0f;
constexpr int kAim = 8;
__device__ __forceinline__ float power_of_2(int n) { return __builtin_bit_cast(float, (unsigned)(127 + n) << 23); }
__device__ __forceinline__ int exponent_of(float x) { return (int)(__builtin_bit_cast(unsigned, x) >> 23) - 127; }   // x >= 0; 128 for infinity

// Waits for every load issued so far.  Called in front of a loop that keeps loads in flight: a register loaded before the loop would otherwise
// be waited for inside it, and the wait for it is a wait for everything.
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0F70); }   // vmcnt(0)

// A row of a tensor straight into operands.  (A column without a query reads the first one's row: nothing of it is stored.)
template <typename T, int DP>
__device__ __forceinline__ void load_frags(const T *p, const AttArgs &a, typename Vec<T>::type (&f)[DP / 16]) {
  const int hi = (threadIdx.x & 63) >> 5;
  if (a.D == DP) {
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) __builtin_memcpy(&f[s], p + 16 * s + 8 * hi, 16);
  } else {
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      const u32x4 r = load16(p + 16 * s + 8 * hi, a.D - 16 * s - 8 * hi);
      __builtin_memcpy(&f[s], &r, 16);
    }
  }
}

// key / per: the quotient in 64 bits is off by one at most, and put right
__device__ __forceinline__ int group_of(const AttArgs &a, int key) {
  int g = (int)(key * a.per_inverse);
  const int rest = key - g * a.per;
  return rest < 0 ? g - 1 : rest >= a.per ? g + 1 : g;
}

// which of a tile's keys are there, one bit each
__device__ __forceinline__ unsigned long long tile_keys(const AttArgs &a, int b, int tile) {
  const int key = tile * kTile + (threadIdx.x & 63);
  bool on = key < a.Lk;
  if (a.keep && on) on = a.keep[(int64_t)b * a.groups + group_of(a, key)] != 0;
  return __ballot(on);
}

__device__ __forceinline__ unsigned long long uniform(unsigned long long m) {
  return (unsigned long long)__builtin_amdgcn_readfirstlane((int)(m >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)m);
}

// Walks the tiles [first, last) of one object that hold a kept key, two buffers in turn.  The work on a tile comes in two halves, step(buffer, keys, 0)
// and (.., 1); beside the first the next tile's k is on its way, beside the second its v (one set of registers for both), each stored into
// the other buffer afterwards.  both(tile, keys) brings a first tile into buffer 0.  All waves make the same calls.
template <typename Both, typename Load, typename Store, typename Step>
__device__ __forceinline__ void walk_tiles(const AttArgs &a, int b, int first, int last, Both both, Load load, Store store, Step step) {
  __shared__ unsigned long long masks[64];
  const int wave = threadIdx.x >> 6;
  for (int c0 = first; c0 < last; c0 += 64) {
    const int n = last - c0 < 64 ? last - c0 : 64;
    for (int i = wave; i < n; i += kWaves) {
      const unsigned long long m = tile_keys(a, b, c0 + i);
      if ((threadIdx.x & 63) == 0) masks[i] = m;
    }
    lds_barrier();
    int i = 0, buffer = 0;
    while (i < n && !masks[i]) ++i;
    unsigned long long m = i < n ? uniform(masks[i]) : 0;
    if (i < n) both(c0 + i, m);
    loads_done();
    lds_barrier();
    while (i < n) {
      int next = i + 1;
      while (next < n && !masks[next]) ++next;
      const unsigned long long mn = next < n ? uniform(masks[next]) : 0;
      if (next < n) load(0, c0 + next);
      step(buffer, m, 0);
      if (next < n) {
        store(0, buffer ^ 1, mn);
        load(1, c0 + next);
      }
      step(buffer, m, 1);
      buffer ^= 1;
      if (next < n) store(1, buffer, mn);
      lds_barrier();
      i = next, m = mn;
    }
  }
}

// what walk_tiles is told for tiles of k and v
#define MVR_ATT_KV                                                                                                      \
  [&](int tile, unsigned long long m) {                                                                                 \
    Stage<T, DP> more;                                                                                                  \
    load_tile<WHOLE>(staged, kb, a.ks[1], tile, a);                                                                            \
    load_tile<WHOLE>(more, vb, a.vs[1], tile, a);                                                                              \
    staged.store(tiles[0], m), more.store(tiles[0] + kSize, m);                                                         \
  },                                                                                                                    \
      [&](int which, int tile) { load_tile<WHOLE>(staged, which ? vb : kb, which ? a.vs[1] : a.ks[1], tile, a); },             \
      [&](int which, int buffer, unsigned long long m) { staged.store(tiles[buffer] + which * kSize, m); }

template <bool WHOLE, typename T, int DP>
__device__ __forceinline__ void load_tile(Stage<T, DP> &staged, const T *base, int64_t stride, int tile, const AttArgs &a) {
  const int at = tile * kTile, left = a.Lk - at;
  base += at * stride;
  if constexpr (WHOLE) staged.load(base, (unsigned)stride, a.D, left < kTile ? left - 1 : kTile - 1);
  else staged.load_rows(a.D, [&](int r) { return r < left ? base + r * stride : nullptr; });
}

// ---- forward -----------------------------------------------------------------------------------------------------

// A lane's column: the query (of one of the group's heads) that it works for
struct Column {
  int64_t row;
  int g, i;
  bool live;
};
__device__ __forceinline__ Column column_of(const AttArgs &a, int ct, int n, int per_wave) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Column c;
  c.row = ((int64_t)ct * kWaves + wave) * per_wave + 32 * n + (lane & 31);
  c.live = c.row < a.rows;
  c.g = c.live ? (int)((unsigned)c.row / (unsigned)a.Lq) : 0;
  c.i = c.live ? (int)c.row - c.g * a.Lq : 0;
  return c;
}
// a column's 32 db values, four by four in the order of the matrix instruction's result
template <typename U, int DP>
__device__ __forceinline__ void store_column(U *p, int D, const f32x16 (&x)[DP / 32], float f) {
  const int hi = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int at = 32 * d + 8 * r + 4 * hi;
      const float v[4] = {x[d][4 * r] * f, x[d][4 * r + 1] * f, x[d][4 * r + 2] * f, x[d][4 * r + 3] * f};
      store_n<4>(p + at, D == DP ? 4 : D - at, v);
    }
}
// what store_column's rounding leaves of the same values
template <typename T, int DP>
__device__ __forceinline__ void store_column_rest(T *p, int D, const f32x16 (&x)[DP / 32], float f) {
  f32x16 y[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) y[d][r] = x[d][r] * f - (float)(T)(x[d][r] * f);
  store_column<T, DP>(p, D, y, 1.0f);
}
// the scores of keys that are not there, replaced: a register's 32 + 32 lanes hold two keys, so their bits make its lane mask on the scalar unit
__device__ __forceinline__ void mask_scores(f32x16 &s, unsigned long long m, int t, float by) {
  const unsigned bits = (unsigned)(m >> (32 * t));
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int at = 8 * (r / 4) + r % 4;
    const unsigned lo = bits >> at & 1 ? ~0u : 0u, hi = bits >> (at + 4) & 1 ? ~0u : 0u;
    s[r] = __builtin_amdgcn_inverse_ballot_w64((unsigned long long)hi << 32 | lo) ? s[r] : by;
  }
}

// The running maximum only has to keep exponentials in range: it follows the scores when one exceeds it by more than kSlack (powers of two),
// and only then are sum and output rescaled.  Probabilities then reach 2^8 (2^15 in float16, with kLift: half its largest number), and their rounding is relative.
// (Following every new maximum, one of a wave's 64 columns has one in four tiles of five, at 68 multiplications each.)
constexpr float kSlack = 8.0f;

// LSE: the sum is also taken of the probabilities as they are, for lse: the backward's P would all be off by what rounding made of the sum, which
// one large probability among them decides.  The output is divided by the sum of the rounded ones, which cancels that.  (Splits are weighted by lse.)
// With `rest` the backward also has the output in more bits than its store: delta = rowsum(dO O) stands against dP, and where one probability is near 1
// the difference is small.  Error of dQ over its store's alone, 1024 keys of 64, scores with a deviation of 1 / 3 / 6 / 10: 1.4 / 1.5 / 1.5 / 1.5 times, without
// the two 1.4 / 1.9 / 2.5 / 3.1.  Forward and gradients with and without: 16 x 2352 tokens, 12 heads of 64, a quarter dropped, 1450 / 1407 us; 8 x 3920, 16
// heads of 128, 5605 / 5520; 16 x 1000, 12 heads of 32 (the forward on two waves a SIMD in place of three) 210 / 196.
//
// FINE (here and in the backward), where all keys lie in one tile: P and dS enter their products, and P the sum, as two parts, a rounded value and what
// its rounding left, and delta comes from P and dP in 32 bits.  Otherwise the gradients carry, beside the store's rounding, one of P and dS (1.4
// times the store's error alone), and in dQ that of P in delta (to 1.5 where few keys have the sum; 1.0 with FINE).  It costs, forward / backward: 384 x 64 tokens, 12 heads of 64 on 4
// 30.4 -> 31.6 / 76 -> 87 us; 16 heads of 128 107 -> 109 / 292 us both; 64 x 1000 queries over 48 keys 60.7 -> 65 / 164 -> 179 us.
//
// NS columns of 32 queries a wave: with two, every operand read from LDS serves two products, and one's exponentials run beside the other's
// products
template <typename T, int DP, int NS, bool SPLIT, bool WHOLE, bool FINE, bool LSE>
__global__ __launch_bounds__(kBlock, 2) void k_attend(AttArgs a) {
  typedef typename Vec<T>::type V8;
  constexpr int kSize = Layout<DP>::kSize;
  __shared__ __attribute__((aligned(256))) T tiles[2][2 * kSize];   // two buffers of a tile of k and a tile of v
  int64_t item = work_item(a.work);
  if (item >= a.work) return;
  const int split = SPLIT ? (int)(item % a.splits) : 0;
  if (SPLIT) item /= a.splits;
  const int ct = (int)(item % a.col_tiles);
  const int64_t be = item / a.col_tiles;
  const int b = (int)(be / a.E), e = (int)(be - (int64_t)b * a.E);
  V8 q[NS][DP / 16];
  f32x16 o[NS][DP / 32];
  float top[NS], sum[NS], sum_as_is[NS];   // of this lane's column; the sums over the rows this lane holds
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    const Column c = column_of(a, ct, n, 32 * NS);
    load_frags<T, DP>((const T *)a.q + b * a.qs[0] + c.i * a.qs[1] + (e * a.G + c.g) * a.qs[2], a, q[n]);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) o[n][d] = 0.0f;
    top[n] = -INFINITY, sum[n] = sum_as_is[n] = 0.0f;
  }
  const T *kb = (const T *)a.k + b * a.ks[0] + e * a.ks[2], *vb = (const T *)a.v + b * a.vs[0] + e * a.vs[2];
  Stage<T, DP> staged;
  const Reader<DP> reader = Reader<DP>::wide(tiles);
  const int first = SPLIT ? split * a.split_tiles : 0, last = SPLIT && first + a.split_tiles < a.tiles ? first + a.split_tiles : a.tiles;
  f32x16 s[NS][2];
  const auto step = [&](int buffer, unsigned long long m, int half) {
    const Reader<DP> r = reader.at(buffer);
    if (half == 1) {   // probabilities and their product with v
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        V8 v[2][DP / 32], p[NS][2];
        col_frags<T, DP>(r, 1, t, v);
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          const float off = top[n] == -INFINITY ? 0.0f : top[n] - kLift<T>;
#pragma unroll
          for (int r = 0; r < 16; ++r) s[n][t][r] = __builtin_amdgcn_exp2f(fmaf(s[n][t][r], a.c, -off));
          if constexpr (LSE) {
#pragma unroll
            for (int r = 0; r < 16; ++r) sum_as_is[n] += s[n][t][r];
          }
          p[n][0] = to_frag<T>(s[n][t], 0), p[n][1] = to_frag<T>(s[n][t], 1);
          sum[n] = add_frag(p[n][1], add_frag(p[n][0], sum[n]));   // (of the probabilities as they enter the product)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) o[n][d] = mfma(v[h][d], p[n][h], o[n][d]);
          if constexpr (FINE) {
            const V8 rest[2] = {rest_frag<T>(s[n][t], 0), rest_frag<T>(s[n][t], 1)};
            sum[n] = add_frag(rest[1], add_frag(rest[0], sum[n]));
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int d = 0; d < DP / 32; ++d) o[n][d] = mfma(v[h][d], rest[h], o[n][d]);
          }
        }
      }
      return;
    }
    // scores, running maximum
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      V8 k[DP / 16];
      row_frags<T, DP>(r, 0, t, k);
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        s[n][t] = 0.0f;
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) s[n][t] = mfma(k[d], q[n][d], s[n][t]);
      }
    }
    if (m != ~0ull) {
#pragma unroll
      for (int n = 0; n < NS; ++n) mask_scores(s[n][0], m, 0, -INFINITY), mask_scores(s[n][1], m, 1, -INFINITY);
    }
    float now[NS];
    bool up = false;
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      float mx = fmaxf(s[n][0][0], s[n][1][0]);
#pragma unroll
      for (int r = 1; r < 16; ++r) mx = fmaxf(fmaxf(s[n][0][r], s[n][1][r]), mx);
      mx = fmaxf(mx, other_half(mx));
      now[n] = fmaxf(top[n], mx * a.c);
      up = up || now[n] > top[n] + kSlack;
    }
    if (__any(up)) {
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        const float f = __builtin_amdgcn_exp2f(top[n] - (now[n] == -INFINITY ? 0.0f : now[n]));
        sum[n] *= f, sum_as_is[n] *= f;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) o[n][d] *= f;
        top[n] = now[n];
      }
    }
  };
  walk_tiles(a, b, first, last, MVR_ATT_KV, step);
  const int hi = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    const Column c = column_of(a, ct, n, 32 * NS);
    const float all = sum[n] + other_half(sum[n]), as_is = LSE ? sum_as_is[n] + other_half(sum_as_is[n]) : all;
    if (!c.live) continue;
    const float inv = all > 0.0f ? 1.0f / all : all == 0.0f ? 0.0f : all;   // (a NaN stays one)
    if constexpr (SPLIT) {
      const int64_t line = (split * (int64_t)a.B * a.E + be) * a.rows + c.row;
      store_column<float, DP>(a.part + line * a.D, a.D, o[n], inv);
      if (hi == 0) a.part_lse[line] = all == 0.0f ? -INFINITY : top[n] - kLift<T> + __builtin_amdgcn_logf(as_is);
    } else {
      const int64_t to = (((int64_t)b * a.Lq + c.i) * a.H + e * a.G + c.g) * a.D;
      store_column<T, DP>((T *)a.out + to, a.D, o[n], inv);
      if constexpr (LSE) {
        if (a.rest) store_column_rest<T, DP>((T *)a.rest + to, a.D, o[n], inv);
      }
      if (a.lse && hi == 0) a.lse[be * a.rows + c.row] = all == 0.0f ? INFINITY : top[n] - kLift<T> + __builtin_amdgcn_logf(as_is);
    }
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
  const int64_t to = ((b * a.Lq + i) * a.H + e * a.G + g) * a.D;
  for (int k = 0; k < 2; ++k)
    if (lane + 64 * k < a.D) {
      const T y = (T)(x[k] * inv);
      ((T *)a.out)[to + lane + 64 * k] = y;
      if (a.rest) ((T *)a.rest)[to + lane + 64 * k] = (T)(x[k] * inv - (float)y);
    }
  if (a.lse && lane == 0) a.lse[line] = sum == 0.0f ? INFINITY : off + __builtin_amdgcn_logf(sum);
}

// ---- dQ (and delta) ----------------------------------------------------------------------------------------------

// One column of 32 queries a wave: with heads of 64 160 registers and three waves a SIMD, where two columns take 246 and leave two.
// 16 x 2352 tokens, 12 heads of 64, 12 views of which a quarter is dropped, bfloat16: 424 us against 472 with two; the forward, which keeps less
// per column, takes 364 us with two and 411 with one.
template <typename T, int DP, bool SPLIT, bool WHOLE, bool FINE>
__global__ __launch_bounds__(kBlock, 2) void k_attend_dq(AttArgs a) {
  typedef typename Vec<T>::type V8;
  constexpr int kSize = Layout<DP>::kSize;
  __shared__ __attribute__((aligned(256))) T tiles[2][2 * kSize];   // two buffers of a tile of k and a tile of v
  int64_t item = work_item(a.work);
  if (item >= a.work) return;
  const int split = SPLIT ? (int)(item % a.splits) : 0;
  if (SPLIT) item /= a.splits;
  const int ct = (int)(item % a.col_tiles);
  const int64_t be = item / a.col_tiles;
  const int b = (int)(be / a.E), e = (int)(be - (int64_t)b * a.E);
  V8 q[DP / 16], go[DP / 16];
  f32x16 dq[DP / 32];
  const Column c = column_of(a, ct, 0, 32);
  const int h = e * a.G + c.g;
  float lse, delta = 0.0f;
  float power = kNarrow<T> ? kStart : 0.0f;   // log2 of what this column's dS and dq are multiplied by (it goes into P's exponent)
  load_frags<T, DP>((const T *)a.q + b * a.qs[0] + c.i * a.qs[1] + h * a.qs[2], a, q);
  load_frags<T, DP>((const T *)a.go + b * a.gs[0] + c.i * a.gs[1] + h * a.gs[2], a, go);
  if constexpr (!FINE) {
    const int64_t at = (((int64_t)b * a.Lq + c.i) * a.H + h) * a.D;
    const auto add = [&](const void *part) {
      V8 o[DP / 16];
      load_frags<T, DP>((const T *)part + at, a, o);
#pragma unroll
      for (int s = 0; s < DP / 16; ++s)
#pragma unroll
        for (int k = 0; k < 8; ++k) delta += (float)o[s][k] * (float)go[s][k];
    };
    add(a.o);
    if (a.rest) add(a.rest);
    delta += other_half(delta);
  }
  lse = c.live ? a.lse[be * a.rows + c.row] : INFINITY;
  const bool writes = c.live && (threadIdx.x & 32) == 0 && split == 0;
  if (!FINE && writes) a.delta[be * a.rows + c.row] = delta;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) dq[d] = 0.0f;
  const T *kb = (const T *)a.k + b * a.ks[0] + e * a.ks[2], *vb = (const T *)a.v + b * a.vs[0] + e * a.vs[2];
  Stage<T, DP> staged;
  const Reader<DP> reader = Reader<DP>::wide(tiles);
  const int first = SPLIT ? split * a.split_tiles : 0, last = SPLIT && first + a.split_tiles < a.tiles ? first + a.split_tiles : a.tiles;
  const auto step = [&](int buffer, unsigned long long m, int t) {
    const Reader<DP> r = reader.at(buffer);
    V8 f[DP / 16], kc[2][DP / 32];
    if (FINE && t == 0) {   // delta over the one tile
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        f32x16 s = 0.0f, dp = 0.0f;
        row_frags<T, DP>(r, 0, u, f);
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) s = mfma(f[d], q[d], s);
        fence();
        row_frags<T, DP>(r, 1, u, f);
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) dp = mfma(f[d], go[d], dp);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -lse));
        if (m != ~0ull) mask_scores(s, m, u, 0.0f);
#pragma unroll
        for (int r = 0; r < 16; ++r) delta = fmaf(s[r], dp[r], delta);
        fence();
      }
      delta += other_half(delta);
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) dq[d] = 0.0f;   // (the zeros from before need no registers until here)
    }
    f32x16 s = 0.0f, dp = 0.0f;
    row_frags<T, DP>(r, 0, t, f);
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) s = mfma(f[d], q[d], s);
    fence();
    row_frags<T, DP>(r, 1, t, f);
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) dp = mfma(f[d], go[d], dp);
    fence();
    if (DP <= 64) col_frags<T, DP>(r, 0, t, kc);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, kNarrow<T> ? power - lse : -lse));
    if (m != ~0ull) mask_scores(s, m, t, 0.0f);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] *= dp[r] - delta;
    if constexpr (kNarrow<T>) {
      float most = 0.0f;
#pragma unroll
      for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(s[r]));
      if (__any(most > kMost)) {
        most = fmaxf(most, other_half(most));
        const int down = most > kMost ? exponent_of(most) - kAim : 0;
        const float by = power_of_2(-down);
        s *= by;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) dq[d] *= by;
        power -= (float)down;
      }
    }
    const V8 ds[2] = {to_frag<T>(s, 0), to_frag<T>(s, 1)};
    V8 rest[2];
    if constexpr (FINE) rest[0] = rest_frag<T>(s, 0), rest[1] = rest_frag<T>(s, 1);
    if (DP > 64) {   // (the scores have been used up: their registers take the operands)
      fence();
      col_frags<T, DP>(r, 0, t, kc);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) {
        dq[d] = mfma(kc[h][d], ds[h], dq[d]);
        if constexpr (FINE) dq[d] = mfma(kc[h][d], rest[h], dq[d]);
      }
    fence();
  };
  walk_tiles(a, b, first, last, MVR_ATT_KV, step);
  if (FINE && writes) a.delta[be * a.rows + c.row] = delta;
  if (c.live) {
    const float back = kNarrow<T> ? __builtin_ldexpf(1.0f, -(int)power) : 1.0f;
    if constexpr (SPLIT) store_column<float, DP>(a.part + ((split * (int64_t)a.B * a.E + be) * a.rows + c.row) * a.D, a.D, dq, back);
    else store_column<T, DP>((T *)a.dq + (((int64_t)b * a.Lq + c.i) * a.H + e * a.G + c.g) * a.D, a.D, dq, a.scale * back);
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
//
// Heads above 64: a column of 16 keys a wave on v_mfma_f32_16x16x32, whose two sums of 16 x D leave the registers for two waves a SIMD, where 32
// keys of 128 fill all of one.  A lane's scores are rows 16 b + 4 (lane / 16) + 0..3 of a sub-tile of 32 (b = 0, 1) of ONE key, which is the order
// that the next product's operands take the rows in.
//
// Few keys: the rows are dealt to several workgroups, as the keys are in the other kernels, and their parts of dK and dV, in 32 bits, are added
// up by k_attend_dkv_join.  4000 queries, 4 heads of 128 on one, forward and gradients, us without and with: over 12 keys (where one workgroup walked 250
// tiles) 569 / 84, over 4000 keys 590 / 248.

__device__ __forceinline__ int64_t dkv_size(const AttArgs &a) { return (int64_t)a.B * a.Lk * a.E * a.D; }

template <typename T, int DP, bool WHOLE, bool FINE>
__global__ __launch_bounds__(kBlock, 2) void k_attend_dkv16(AttArgs a) {
  typedef typename Vec<T>::type V8;
  typedef Reader<DP> R;
  constexpr int kSize = Layout<DP>::kSize;
  __shared__ __attribute__((aligned(256))) T tiles[2][2 * kSize];   // two buffers of a tile of q and a tile of dO
  __shared__ __attribute__((aligned(16))) float stats[2][2][kTile];   // their lse and -delta
  int64_t item = work_item(a.work);
  if (item >= a.work) return;
  const int split = (int)(item % a.row_splits);
  item /= a.row_splits;
  const int ct = (int)(item % a.col_tiles);
  const int64_t be = item / a.col_tiles;
  const int b = (int)(be / a.E), e = (int)(be - (int64_t)b * a.E);
  const int wave = threadIdx.x >> 6;
  const R reader = R::narrow(tiles);
  V8 k[DP / 32], v[DP / 32];
  f32x4 dk[DP / 16], dv[DP / 16];
  const int lane = threadIdx.x & 63, key = (ct * kWaves + wave) * 16 + (lane & 15);
  const bool there = key < a.Lk, on = there && (!a.keep || a.keep[(int64_t)b * a.groups + group_of(a, key)] != 0);
  const T *pk = (const T *)a.k + b * a.ks[0] + (int64_t)key * a.ks[1] + e * a.ks[2], *pv = (const T *)a.v + b * a.vs[0] + (int64_t)key * a.vs[1] + e * a.vs[2];
#pragma unroll
  for (int s = 0; s < DP / 32; ++s) {
    const int at = 32 * s + 8 * (lane >> 4);
    const u32x4 x = load16(pk + at, on ? a.D - at : 0), y = load16(pv + at, on ? a.D - at : 0);
    __builtin_memcpy(&k[s], &x, 16), __builtin_memcpy(&v[s], &y, 16);
  }
#pragma unroll
  for (int d = 0; d < DP / 16; ++d) dk[d] = 0.0f, dv[d] = 0.0f;
  const bool all = __all(on);
  const T *qb = (const T *)a.q + b * a.qs[0] + (int64_t)e * a.G * a.qs[2], *gb = (const T *)a.go + b * a.gs[0] + (int64_t)e * a.G * a.gs[2];
  Stage<T, DP> staged;
  float lse = 0.0f, delta = 0.0f;
  float times = power_of_2((int)kStart);   // what this column's dS and dk are multiplied by (kNarrow)
  const int head_tiles = (a.Lq + kTile - 1) / kTile, all_tiles = WHOLE ? a.G * head_tiles : (a.rows + kTile - 1) / kTile;
  const int first = split * a.row_split_tiles, end = first + a.row_split_tiles < all_tiles ? first + a.row_split_tiles : all_tiles;
  const int n = __syncthreads_or(on) ? end : first;   // (no kept key here: zeros)
  // as in walk_tiles: a tile of q beside the first half of the work, a tile of dO beside the second
  // the tile to load: with WHOLE from row i0 of head g0 (a head's last tile ends with it), else the rows from tile * kTile of the group's list
  int g0 = WHOLE ? first / head_tiles : 0, i0 = WHOLE ? (first - g0 * head_tiles) * kTile : 0;
  const auto load = [&](int which, int tile) {
    const T *base = which ? gb : qb;
    const int64_t stride = which ? a.gs[1] : a.qs[1], head = which ? a.gs[2] : a.qs[2];
    const int at = WHOLE ? g0 * a.Lq + i0 : tile * kTile, left = (WHOLE ? a.Lq - i0 : a.rows - at);
    if constexpr (WHOLE) {
      staged.load(base + (int64_t)i0 * stride + g0 * head, (unsigned)stride, a.D, left < kTile ? left - 1 : kTile - 1);
    } else {
      staged.load_rows(a.D, [&](int r) -> const T * {
        const int row = at + r, g = row / a.Lq;
        return r < left ? base + (int64_t)(row - g * a.Lq) * stride + g * head : nullptr;
      });
    }
    if (which == 0 && threadIdx.x < kTile) {
      const bool in = (int)threadIdx.x < left;
      const int64_t row = be * a.rows + at + (in ? threadIdx.x : 0);
      const float x = a.lse[row], y = a.delta[row];
      lse = in ? x : INFINITY, delta = y;   // (behind the last row: probabilities of 0)
    }
    if (WHOLE && which == 1 && (i0 += kTile) >= a.Lq) i0 = 0, ++g0;
  };
  const auto store = [&](int which, int buffer) {
    staged.store(tiles[buffer] + which * kSize, ~0ull);
    if (which == 0 && threadIdx.x < kTile) stats[buffer][0][threadIdx.x] = lse - kLiftP<T>, stats[buffer][1][threadIdx.x] = -delta;
  };
  if (first < n) {
    load(0, first);
    store(0, 0);
    load(1, first);
    store(1, 0);
  }
  loads_done();
  lds_barrier();
  for (int tile = first; tile < n; ++tile) {
    const int buffer = (tile - first) & 1;
    const R r = reader.at(buffer);
    if (tile + 1 < n) load(0, tile + 1);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if (!WHOLE && t == 1 && a.rows - tile * kTile <= 32) break;   // the list's last tile: no rows in its second half (64 x 4 rows over 3920 keys of 128: 273 -> 262 us)
      f32x4 s[2], dp[2];
      V8 p, ds, p_rest, ds_rest;   // (the rests with FINE alone)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[h] = 0.0f;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
          const V8 f = R::template load<V8>((r.row ^ 64 * d) + (32 * t + 16 * h) * R::kRow);
          s[h] = mfma16(f, k[d], s[h]);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4 from = *reinterpret_cast<const f32x4 *>(&stats[buffer][1][32 * t + 16 * h + 4 * (lane >> 4)]);   // dO v^T starts from -delta
        dp[h] = from;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
          const V8 f = R::template load<V8>((r.row ^ 64 * d) + R::kBytes + (32 * t + 16 * h) * R::kRow);
          dp[h] = mfma16(f, v[d], dp[h]);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4 l = *reinterpret_cast<const f32x4 *>(&stats[buffer][0][32 * t + 16 * h + 4 * (lane >> 4)]);
#pragma unroll
        for (int r = 0; r < 4; ++r) s[h][r] = __builtin_amdgcn_exp2f(fmaf(s[h][r], a.c, -l[r]));
        if (!all) {
#pragma unroll
          for (int r = 0; r < 4; ++r) s[h][r] = on ? s[h][r] : 0.0f;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[4 * h + r] = (T)s[h][r];
          if constexpr (FINE) p_rest[4 * h + r] = (T)(s[h][r] - (float)p[4 * h + r]);
          dp[h][r] *= s[h][r];
        }
      }
      if constexpr (kNarrow<T>) {
        float most = 0.0f;
#pragma unroll
        for (int r = 0; r < 8; ++r) most = fmaxf(most, fabsf(dp[r / 4][r % 4]));
        if (__any(most * times > kMost)) {
          most = fmaxf(most, __shfl_xor(most, 16)), most = fmaxf(most, __shfl_xor(most, 32));
          const float now = most * times > kMost ? power_of_2(kAim - exponent_of(most)) : times;
#pragma unroll
          for (int d = 0; d < DP / 16; ++d) dk[d] *= now / times;
          times = now;
        }
        dp[0] *= times, dp[1] *= times;
      }
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        ds[r] = (T)dp[r / 4][r % 4];
        if constexpr (FINE) ds_rest[r] = (T)(dp[r / 4][r % 4] - (float)ds[r]);
      }
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) {
        const V8 f = R::template load_columns<V8>((r.col ^ 32 * d) + R::kBytes + 32 * t * R::kRow, (r.col ^ 32 * d) + R::kBytes + (32 * t + 16) * R::kRow);
        dv[d] = mfma16(f, p, dv[d]);
        if constexpr (FINE) dv[d] = mfma16(f, p_rest, dv[d]);
      }
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) {
        const V8 f = R::template load_columns<V8>((r.col ^ 32 * d) + 32 * t * R::kRow, (r.col ^ 32 * d) + (32 * t + 16) * R::kRow);
        dk[d] = mfma16(f, ds, dk[d]);
        if constexpr (FINE) dk[d] = mfma16(f, ds_rest, dk[d]);
      }
      if (tile + 1 < n) {
        store(t, buffer ^ 1);
        if (t == 0) load(1, tile + 1);
      }
    }
    lds_barrier();
  }
  if (!there) return;
  if (!on) {   // (P = 0 times what dO or q hold is not 0 where they hold infinities)
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) dk[d] = dv[d] = 0.0f;
  }
  const int64_t to = (((int64_t)b * a.Lk + key) * a.E + e) * a.D;
  const float scale = a.row_splits > 1 ? 1.0f : a.scale;   // (parts are scaled where they are added up)
  const float dv_by = kNarrow<T> ? power_of_2(-(int)kLiftP<T>) : 1.0f, dk_by = kNarrow<T> ? scale * dv_by / times : scale;
  float *part = a.part + split * 2 * dkv_size(a) + to;
#pragma unroll
  for (int d = 0; d < DP / 16; ++d) {
    const int at = 16 * d + 4 * (lane >> 4);
    const float x[4] = {dk[d][0] * dk_by, dk[d][1] * dk_by, dk[d][2] * dk_by, dk[d][3] * dk_by};
    const float y[4] = {dv[d][0] * dv_by, dv[d][1] * dv_by, dv[d][2] * dv_by, dv[d][3] * dv_by};
    if (a.row_splits > 1) {
      store_n<4>(part + at, a.D - at, x);
      store_n<4>(part + dkv_size(a) + at, a.D - at, y);
    } else {
      store_n<4>((T *)a.dk + to + at, a.D - at, x);
      store_n<4>((T *)a.dv + to + at, a.D - at, y);
    }
  }
}

// Heads of 64 and less: a column of 32 keys a wave on v_mfma_f32_32x32x16, half the reads of LDS per product
template <typename T, int DP, bool WHOLE, bool FINE>
__global__ __launch_bounds__(kBlock, 2) void k_attend_dkv32(AttArgs a) {
  typedef typename Vec<T>::type V8;
  constexpr int kSize = Layout<DP>::kSize;
  __shared__ __attribute__((aligned(256))) T tiles[2][2 * kSize];   // two buffers of a tile of q and a tile of dO
  __shared__ __attribute__((aligned(16))) float stats[2][2][kTile];   // their lse and -delta
  int64_t item = work_item(a.work);
  if (item >= a.work) return;
  const int split = (int)(item % a.row_splits);
  item /= a.row_splits;
  const int ct = (int)(item % a.col_tiles);
  const int64_t be = item / a.col_tiles;
  const int b = (int)(be / a.E), e = (int)(be - (int64_t)b * a.E);
  const int lane = threadIdx.x & 63, hi = lane >> 5, wave = threadIdx.x >> 6;
  const int key = ct * (32 * kWaves) + wave * 32 + (lane & 31);
  const bool there = key < a.Lk, on = there && (!a.keep || a.keep[(int64_t)b * a.groups + group_of(a, key)] != 0);
  V8 k[DP / 16], v[DP / 16];
  const auto key_frags = [&](const T *p, V8 (&f)[DP / 16]) {
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      const u32x4 r = load16(p + 16 * s + 8 * hi, on ? a.D - 16 * s - 8 * hi : 0);
      __builtin_memcpy(&f[s], &r, 16);
    }
  };
  key_frags((const T *)a.k + b * a.ks[0] + (int64_t)key * a.ks[1] + e * a.ks[2], k);
  key_frags((const T *)a.v + b * a.vs[0] + (int64_t)key * a.vs[1] + e * a.vs[2], v);
  const bool all = __all(on);
  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) dk[d] = 0.0f, dv[d] = 0.0f;
  const T *qb = (const T *)a.q + b * a.qs[0] + (int64_t)e * a.G * a.qs[2], *gb = (const T *)a.go + b * a.gs[0] + (int64_t)e * a.G * a.gs[2];
  Stage<T, DP> staged;
  const Reader<DP> reader = Reader<DP>::wide(tiles);
  float lse = 0.0f, delta = 0.0f;
  float times = power_of_2((int)kStart);   // what this column's dS and dk are multiplied by (kNarrow)
  const int head_tiles = (a.Lq + kTile - 1) / kTile, all_tiles = WHOLE ? a.G * head_tiles : (a.rows + kTile - 1) / kTile;
  const int first = split * a.row_split_tiles, end = first + a.row_split_tiles < all_tiles ? first + a.row_split_tiles : all_tiles;
  const int n = __syncthreads_or(on) ? end : first;   // (no kept key here: zeros)
  // as in walk_tiles: a tile of q beside the first half of the work, a tile of dO beside the second
  // the tile to load: with WHOLE from row i0 of head g0 (a head's last tile ends with it), else the rows from tile * kTile of the group's list
  int g0 = WHOLE ? first / head_tiles : 0, i0 = WHOLE ? (first - g0 * head_tiles) * kTile : 0;
  const auto load = [&](int which, int tile) {
    const T *base = which ? gb : qb;
    const int64_t stride = which ? a.gs[1] : a.qs[1], head = which ? a.gs[2] : a.qs[2];
    const int at = WHOLE ? g0 * a.Lq + i0 : tile * kTile, left = (WHOLE ? a.Lq - i0 : a.rows - at);
    if constexpr (WHOLE) {
      staged.load(base + (int64_t)i0 * stride + g0 * head, (unsigned)stride, a.D, left < kTile ? left - 1 : kTile - 1);
    } else {
      staged.load_rows(a.D, [&](int r) -> const T * {
        const int row = at + r, g = row / a.Lq;
        return r < left ? base + (int64_t)(row - g * a.Lq) * stride + g * head : nullptr;
      });
    }
    if (which == 0 && threadIdx.x < kTile) {
      const bool in = (int)threadIdx.x < left;
      const int64_t row = be * a.rows + at + (in ? threadIdx.x : 0);
      const float x = a.lse[row], y = a.delta[row];
      lse = in ? x : INFINITY, delta = y;   // (behind the last row: probabilities of 0)
    }
    if (WHOLE && which == 1 && (i0 += kTile) >= a.Lq) i0 = 0, ++g0;
  };
  const auto store = [&](int which, int buffer) {
    staged.store(tiles[buffer] + which * kSize, ~0ull);
    if (which == 0 && threadIdx.x < kTile) stats[buffer][0][threadIdx.x] = lse - kLiftP<T>, stats[buffer][1][threadIdx.x] = -delta;
  };
  if (first < n) {
    load(0, first);
    store(0, 0);
    load(1, first);
    store(1, 0);
  }
  loads_done();
  lds_barrier();
  for (int tile = first; tile < n; ++tile) {
    const int buffer = (tile - first) & 1;
    const Reader<DP> r = reader.at(buffer);
    if (tile + 1 < n) load(0, tile + 1);
    V8 qf[DP / 16], gf[DP / 16], c[2][DP / 32];
    row_frags<T, DP>(r, 0, 0, qf);
    fence();
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if (!WHOLE && t == 1 && a.rows - tile * kTile <= 32) break;   // the list's last tile: no rows in its second half
      f32x16 s = 0.0f, dp, l;
      row_frags<T, DP>(r, 1, t, gf);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float4 x = *reinterpret_cast<const float4 *>(&stats[buffer][1][32 * t + 8 * r + 4 * hi]);
        const float4 y = *reinterpret_cast<const float4 *>(&stats[buffer][0][32 * t + 8 * r + 4 * hi]);
        dp[4 * r] = x.x, dp[4 * r + 1] = x.y, dp[4 * r + 2] = x.z, dp[4 * r + 3] = x.w;
        l[4 * r] = y.x, l[4 * r + 1] = y.y, l[4 * r + 2] = y.z, l[4 * r + 3] = y.w;
      }
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) s = mfma(qf[d], k[d], s);
      fence();
      col_frags<T, DP>(r, 1, t, c);
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) dp = mfma(gf[d], v[d], dp);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -l[r]));
      if (!all) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = on ? s[r] : 0.0f;
      }
      const V8 p[2] = {to_frag<T>(s, 0), to_frag<T>(s, 1)};
      fence();
      V8 c2[2][DP / 32];
      col_frags<T, DP>(r, 0, t, c2);
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
          dv[d] = mfma(c[half][d], p[half], dv[d]);
          if constexpr (FINE) dv[d] = mfma(c[half][d], rest_frag<T>(s, half), dv[d]);
        }
      dp *= s;
      if constexpr (kNarrow<T>) {
        float most = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(dp[r]));
        if (__any(most * times > kMost)) {
          most = fmaxf(most, other_half(most));
          const float now = most * times > kMost ? power_of_2(kAim - exponent_of(most)) : times;
#pragma unroll
          for (int d = 0; d < DP / 32; ++d) dk[d] *= now / times;
          times = now;
        }
        dp *= times;
      }
      const V8 ds[2] = {to_frag<T>(dp, 0), to_frag<T>(dp, 1)};
      fence();
      if (t == 0) row_frags<T, DP>(r, 0, 1, qf);
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
          dk[d] = mfma(c2[half][d], ds[half], dk[d]);
          if constexpr (FINE) dk[d] = mfma(c2[half][d], rest_frag<T>(dp, half), dk[d]);
        }
      fence();
      if (tile + 1 < n) {
        store(t, buffer ^ 1);
        if (t == 0) load(1, tile + 1);
      }
    }
    lds_barrier();
  }
  if (!there) return;
  if (!on) {   // (as above)
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) dk[d] = dv[d] = 0.0f;
  }
  const int64_t to = (((int64_t)b * a.Lk + key) * a.E + e) * a.D;
  const float scale = a.row_splits > 1 ? 1.0f : a.scale;   // (as above)
  const float dv_by = kNarrow<T> ? power_of_2(-(int)kLiftP<T>) : 1.0f, dk_by = kNarrow<T> ? scale * dv_by / times : scale;
  if (a.row_splits > 1) {
    float *part = a.part + split * 2 * dkv_size(a) + to;
    store_column<float, DP>(part, a.D, dk, dk_by);
    store_column<float, DP>(part + dkv_size(a), a.D, dv, dv_by);
  } else {
    store_column<T, DP>((T *)a.dk + to, a.D, dk, dk_by);
    store_column<T, DP>((T *)a.dv + to, a.D, dv, dv_by);
  }
}

// one wave per key and head: the parts of the rows' splits, in order
template <typename T>
__global__ __launch_bounds__(kBlock) void k_attend_dkv_join(AttArgs a) {
  const int64_t lines = (int64_t)a.B * a.Lk * a.E, line = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (line >= lines) return;
  const int lane = threadIdx.x & 63;
  for (int k = 0; k < 2; ++k) {
    const int64_t at = line * a.D + lane + 64 * k;
    if (lane + 64 * k >= a.D) break;
    float x = 0.0f, y = 0.0f;
    for (int s = 0; s < a.row_splits; ++s) x += a.part[2 * s * dkv_size(a) + at], y += a.part[(2 * s + 1) * dkv_size(a) + at];
    ((T *)a.dk)[at] = (T)(x * a.scale);
    ((T *)a.dv)[at] = (T)y;
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------

// keys of a workgroup of dK and dV
constexpr int dkv_keys(int D) { return D <= 64 ? 32 * kWaves : 16 * kWaves; }

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
  a.per_inverse = 1.0 / a.per;
  a.scale = p->scale, a.c = p->scale * 1.44269504088896340736f;
  for (int k = 0; k < 3; ++k) a.qs[k] = p->q_stride[k], a.ks[k] = p->k_stride[k], a.vs[k] = p->v_stride[k], a.gs[k] = p->grad_stride[k];
  a.tiles = (p->keys + kTile - 1) / kTile;
  a.whole = p->dim % 8 == 0;
  for (const int64_t *t : {a.qs, a.ks, a.vs, a.gs}) a.whole = a.whole && t[1] >= 0 && t[1] < 1 << 24;
  // two columns of 32 queries a wave where heads leave the registers for it and there are queries enough
  a.wide = a.whole && p->dim <= 64 && rows > 32 * kWaves;
  // few columns: the keys are dealt to several workgroups until there are about two per CU, each with four tiles at least
  const int64_t per = 32 * kWaves * (1 + a.wide), cols = (rows + per - 1) / per, blocks = cols * a.B * a.E;
  int64_t splits = 512 / blocks, most = a.tiles / 4;
  splits = splits > most ? most : splits;
  a.splits = splits < 2 ? 1 : (int32_t)splits;
  a.split_tiles = (a.tiles + a.splits - 1) / a.splits;
  a.splits = (a.tiles + a.split_tiles - 1) / a.split_tiles;
  // few keys: the same for the rows that dK and dV walk
  a.rows_whole = a.whole && (a.G == 1 || a.Lq >= kTile);
  const int64_t row_tiles = a.rows_whole ? (int64_t)a.G * ((a.Lq + kTile - 1) / kTile) : (rows + kTile - 1) / kTile;
  const int64_t key_blocks = (a.Lk + dkv_keys(a.D) - 1) / dkv_keys(a.D) * a.B * a.E;
  splits = 512 / key_blocks, most = row_tiles / 4;
  splits = splits > most ? most : splits;
  a.row_splits = splits < 2 ? 1 : (int32_t)splits;
  a.row_split_tiles = (int32_t)((row_tiles + a.row_splits - 1) / a.row_splits);
  a.row_splits = (int32_t)((row_tiles + a.row_split_tiles - 1) / a.row_split_tiles);
  return MVR_OK;
}

size_t lines(const AttArgs &a) { return (size_t)a.B * a.E * a.rows; }
size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }
size_t forward_bytes(const AttArgs &a) { return a.splits > 1 ? align256(lines(a) * a.splits * a.D * 4) + align256(lines(a) * a.splits * 4) : 0; }
// delta, and the parts of dQ or, behind them in time, of dK and dV
size_t backward_bytes(const AttArgs &a) {
  const size_t dq = a.splits > 1 ? lines(a) * a.splits * a.D * 4 : 0, dkv = a.row_splits > 1 ? (size_t)a.B * a.Lk * a.E * a.D * a.row_splits * 2 * 4 : 0;
  return align256(lines(a) * 4) + align256(dq > dkv ? dq : dkv);
}

// workgroups of `per` columns each, a multiple of 8 for work_item
bool grid_of(AttArgs &a, int64_t columns, int per, int splits, unsigned &blocks) {
  a.col_tiles = (int32_t)((columns + per - 1) / per);
  a.work = (int64_t)a.col_tiles * a.B * a.E * splits;
  const int64_t n = (a.work + 7) / 8 * 8;
  blocks = (unsigned)n;
  return n <= 0x7FFFFFFF;
}

template <typename T, int DP, bool SPLIT, bool FINE, bool LSE>
void launch_attend(const AttArgs &a, unsigned n, hipStream_t st) {
  const dim3 g(n), blk(kBlock);
  constexpr int kWide = DP <= 64 ? 2 : 1;
  if (a.wide) hipLaunchKernelGGL((k_attend<T, DP, kWide, SPLIT, true, FINE, LSE>), g, blk, 0, st, a);
  else if (a.whole) hipLaunchKernelGGL((k_attend<T, DP, 1, SPLIT, true, FINE, LSE>), g, blk, 0, st, a);
  else hipLaunchKernelGGL((k_attend<T, DP, 1, SPLIT, false, FINE, LSE>), g, blk, 0, st, a);
}

template <typename T, int DP>
int launch_forward(AttArgs a, hipStream_t st) {
  unsigned n;
  if (!grid_of(a, a.rows, 32 * kWaves * (1 + a.wide), a.splits, n)) return bad("mvr_attend_tokens_forward: too many workgroups");
  if (a.tiles == 1) launch_attend<T, DP, false, true, false>(a, n, st);   // (FINE's sum is the one of P as it is)
  else if (a.splits > 1) launch_attend<T, DP, true, false, true>(a, n, st);
  else if (a.lse) launch_attend<T, DP, false, false, true>(a, n, st);
  else launch_attend<T, DP, false, false, false>(a, n, st);
  if (int rc = launched("k_attend")) return rc;
  if (a.splits == 1) return MVR_OK;
  hipLaunchKernelGGL((k_attend_join<T>), dim3((unsigned)((lines(a) + kWaves - 1) / kWaves)), dim3(kBlock), 0, st, a);
  return launched("k_attend_join");
}

template <typename T, int DP>
int launch_backward(AttArgs a, hipStream_t st) {
  unsigned n;
  if (!grid_of(a, a.rows, 32 * kWaves, a.splits, n)) return bad("mvr_attend_tokens_backward: too many workgroups");
  const bool fine = a.tiles == 1;
  if (fine) {
    if (a.whole) hipLaunchKernelGGL((k_attend_dq<T, DP, false, true, true>), dim3(n), dim3(kBlock), 0, st, a);
    else hipLaunchKernelGGL((k_attend_dq<T, DP, false, false, true>), dim3(n), dim3(kBlock), 0, st, a);
  } else if (a.splits == 1) {
    if (a.whole) hipLaunchKernelGGL((k_attend_dq<T, DP, false, true, false>), dim3(n), dim3(kBlock), 0, st, a);
    else hipLaunchKernelGGL((k_attend_dq<T, DP, false, false, false>), dim3(n), dim3(kBlock), 0, st, a);
  } else {
    if (a.whole) hipLaunchKernelGGL((k_attend_dq<T, DP, true, true, false>), dim3(n), dim3(kBlock), 0, st, a);
    else hipLaunchKernelGGL((k_attend_dq<T, DP, true, false, false>), dim3(n), dim3(kBlock), 0, st, a);
  }
  if (int rc = launched("k_attend_dq")) return rc;
  if (a.splits > 1) {
    hipLaunchKernelGGL((k_attend_dq_join<T>), dim3((unsigned)((lines(a) + kWaves - 1) / kWaves)), dim3(kBlock), 0, st, a);
    if (int rc = launched("k_attend_dq_join")) return rc;
  }
  const bool whole = a.rows_whole;
  if (!grid_of(a, a.Lk, dkv_keys(DP), a.row_splits, n)) return bad("mvr_attend_tokens_backward: too many workgroups");
  const dim3 g(n), blk(kBlock);
#define MVR_ATT_KEYS(kernel)                                                                \
  do {                                                                                      \
    if (fine && whole) hipLaunchKernelGGL((kernel<T, DP, true, true>), g, blk, 0, st, a);   \
    else if (fine) hipLaunchKernelGGL((kernel<T, DP, false, true>), g, blk, 0, st, a);      \
    else if (whole) hipLaunchKernelGGL((kernel<T, DP, true, false>), g, blk, 0, st, a);     \
    else hipLaunchKernelGGL((kernel<T, DP, false, false>), g, blk, 0, st, a);               \
  } while (0)
  if constexpr (DP <= 64) MVR_ATT_KEYS(k_attend_dkv32);
  else MVR_ATT_KEYS(k_attend_dkv16);
#undef MVR_ATT_KEYS
  if (int rc = launched("k_attend_dkv")) return rc;
  if (a.row_splits == 1) return MVR_OK;
  hipLaunchKernelGGL((k_attend_dkv_join<T>), dim3((unsigned)(((int64_t)a.B * a.Lk * a.E + kWaves - 1) / kWaves)), dim3(kBlock), 0, st, a);
  return launched("k_attend_dkv_join");
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

extern "C" int mvr_attend_tokens_forward_rest(const mvr_attend_params *params, const void *q, const void *k, const void *v, const uint8_t *keep, void *out,
                                              void *out_rest, float *lse, void *workspace, size_t workspace_bytes, mvr_stream_t stream) {
  AttArgs a = {};
  if (int rc = att_args(a, params)) return rc;
  if (!q || !k || !v || !out) return bad("mvr_attend_tokens_forward: q, k, v and out must be given");
  if (out == q || out == k || out == v) return bad("mvr_attend_tokens_forward: out must not be an input");
  if (out_rest && !lse) return bad("mvr_attend_tokens_forward: out_rest goes with lse");
  if (out_rest && (out_rest == q || out_rest == k || out_rest == v || out_rest == out)) return bad("mvr_attend_tokens_forward: out_rest must be memory of its own");
  if ((keep != nullptr) != (params->keep_groups > 0)) return bad("mvr_attend_tokens_forward: keep goes with its groups");
  const size_t need = forward_bytes(a);
  if (need && (!workspace || workspace_bytes < need))
    return fail(MVR_ERR_WORKSPACE, "mvr_attend_tokens_forward: the workspace is smaller than mvr_attend_tokens_workspace_bytes says");
  a.q = q, a.k = k, a.v = v, a.keep = keep, a.out = out, a.rest = out_rest, a.lse = lse;
  a.part = (float *)workspace, a.part_lse = (float *)((char *)workspace + align256(lines(a) * a.splits * a.D * 4));
  const hipStream_t st = (hipStream_t)stream;
  return params->type == MVR_TYPE_HALF ? MVR_ATT_DIMS(launch_forward, f16, a, st) : MVR_ATT_DIMS(launch_forward, bf16, a, st);
}

extern "C" int mvr_attend_tokens_forward(const mvr_attend_params *params, const void *q, const void *k, const void *v, const uint8_t *keep, void *out,
                                         float *lse, void *workspace, size_t workspace_bytes, mvr_stream_t stream) {
  return mvr_attend_tokens_forward_rest(params, q, k, v, keep, out, nullptr, lse, workspace, workspace_bytes, stream);
}

extern "C" int mvr_attend_tokens_backward_rest(const mvr_attend_params *params, const void *q, const void *k, const void *v, const uint8_t *keep,
                                               const void *out, const void *out_rest, const float *lse, const void *grad_out, void *grad_q,
                                               void *grad_k, void *grad_v, void *workspace, size_t workspace_bytes, mvr_stream_t stream) {
  AttArgs a = {};
  if (int rc = att_args(a, params)) return rc;
  if (!q || !k || !v || !out || !lse || !grad_out || !grad_q || !grad_k || !grad_v)
    return bad("mvr_attend_tokens_backward: every tensor but keep must be given");
  if ((keep != nullptr) != (params->keep_groups > 0)) return bad("mvr_attend_tokens_backward: keep goes with its groups");
  if (!workspace || workspace_bytes < backward_bytes(a))
    return fail(MVR_ERR_WORKSPACE, "mvr_attend_tokens_backward: the workspace is smaller than mvr_attend_tokens_workspace_bytes says");
  a.q = q, a.k = k, a.v = v, a.keep = keep, a.o = out, a.rest = const_cast<void *>(out_rest), a.lse = const_cast<float *>(lse), a.go = grad_out, a.dq = grad_q, a.dk = grad_k, a.dv = grad_v;
  a.delta = (float *)workspace, a.part = (float *)((char *)workspace + align256(lines(a) * 4));
  const hipStream_t st = (hipStream_t)stream;
  return params->type == MVR_TYPE_HALF ? MVR_ATT_DIMS(launch_backward, f16, a, st) : MVR_ATT_DIMS(launch_backward, bf16, a, st);
}

extern "C" int mvr_attend_tokens_backward(const mvr_attend_params *params, const void *q, const void *k, const void *v, const uint8_t *keep,
                                          const void *out, const float *lse, const void *grad_out, void *grad_q, void *grad_k, void *grad_v,
                                          void *workspace, size_t workspace_bytes, mvr_stream_t stream) {
  return mvr_attend_tokens_backward_rest(params, q, k, v, keep, out, nullptr, lse, grad_out, grad_q, grad_k, grad_v, workspace, workspace_bytes, stream);
}
