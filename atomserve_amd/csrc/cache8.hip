// A paged cache of keys and values in 8 bits, and attention over it.
//
// Pages of one layer hold e4m3 numbers, in blocks of 16 tokens that share a scale for each kv head:
//
//   k_pages  [num_pages, KV, bs, D]            a block of keys: 16 rows of D bytes
//   v_pages  [num_pages, KV, bs / 16, D, 16]   a block of values, transposed: for every coordinate its 16 tokens
//   scales   fp32 [num_pages, KV, bs / 16]     one for the keys and one for the values; a number is its e4m3 value times the scale
//
// A token at position p of a request lives in page table[p / bs] at offset p % bs, so that a block of either kind is 16 D bytes in one piece, at
// the same place in both.  A block's scale is the power of two 2^e with the smallest e in -100 .. 119 for which its largest magnitude is at
// most 448 * 2^e (448 is the largest e4m3 number).  A block is filled token by token while its scale grows, and what it holds is then
// rewritten: times a power of two an e4m3 number stays the same number unless it falls under the smallest normal one, 2^-6 of the scale (2^-14.8 to
// 2^-13.8 of the largest).  So a number above that is what a single rounding gives, off by at most 2^-4 of itself, however its tokens came; one below is
// rounded again at every growth, by half a smallest step of scales that double at least: by at most 2^-9 of the last scale in all.  Integers, or any
// scale, would be rounded anew each time throughout.
#include "attn_parts.h"
#include "wide_tile.h"

#include <algorithm>

namespace {

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

constexpr int BLOCK = 16;                // tokens that share a scale
constexpr int LEAST = -100, MOST = 119;  // a scale's exponent: below, bf16 numbers would be no normal ones; above, 448 times it would be none
constexpr float LARGEST = 448.f;
constexpr float LOG2E = 1.4426950408889634f;

// The scale of numbers of up to `amax` (finite): 448 is 1.75 * 2^8, and a mantissa beyond 1.75 carries into the exponent.
__device__ __forceinline__ float block_scale(float amax) {
  const int e = (int)((__float_as_uint(amax) + 0x1fffffu) >> 23) - 127 - 8;
  return __uint_as_float((unsigned)(min(max(e, LEAST), MOST) + 127) << 23);
}
// 1 / 2^e, exact
__device__ __forceinline__ float inverse_of(float scale) { return __uint_as_float((254u << 23) - __float_as_uint(scale)); }

// Four numbers of at most 448 as e4m3, to the nearest, in a word.
__device__ __forceinline__ unsigned pack4(float a, float b, float c, float d) {
  const int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
__device__ __forceinline__ float at_most_largest(float x) { return __builtin_amdgcn_fmed3f(x, -LARGEST, LARGEST); }
__device__ __forceinline__ unsigned rescale4(unsigned w, float by) {
  const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return pack4(a[0] * by, a[1] * by, b[0] * by, b[1] * by);
}

struct Pages {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  int num_pages, KV, nb;  // nb: blocks of a page
};
__device__ __forceinline__ size_t block_index(const Pages& p, int page, int kvh, int sub) { return ((size_t)page * p.KV + kvh) * p.nb + sub; }

// ---- appending ------------------------------------------------------------------------------------------
//
// A head is D / 8 lanes' work: lane j < R / 8 has the pairs 4 j .. 4 j + 3 of its rotation (coordinates i and i + R/2), the others eight coordinates that
// are not turned; no lane needs another's but for the sum of squares.
//
// Queries: a group of lanes a (token, head), heads side by side.  Keys and values: a wave takes the runs that start among `chunk` neighbouring tokens, for
// one kv head's keys or values; single tokens several at once, longer runs one after the other.  A run: tokens next to each other in the step that go to places next to each other of one block, so that one wave sees
// all that the step puts there: the largest magnitude, the scale, and what the block held.  Lane group s has the run's places PASSES s .. + PASSES - 1 of the
// block, so that a coordinate's bytes are neighbours in a lane's hands: they cross to the transposed block through LDS.
//
// Bound by memory where there is much of it (a prompt of 2,048 tokens, 32 heads of 128 on 8: 11.4 us, 47 MB at 4.2 TB/s; 16-bit pages 12.7) and by a launch
// and three dependent waits (slots, scale, stores) where there is not: one token 3.0 us, 64 requests' tokens 3.8 to 4.0, 2.6 of it the queries.
template <int D> struct Lanes {
  static constexpr int LPT = D <= 64 ? 8 : D <= 128 ? 16 : 32;  // lanes of a head, D / 8 of them busy
  static constexpr int AT_ONCE = WAVE / LPT, PASSES = BLOCK / AT_ONCE;
};

template <int LPT> __device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (LPT >= 32) v = plus_16(v);
  if constexpr (LPT >= 16) v += dpp<DPP_ROTATE(8)>(v);
  v += dpp<DPP_XOR_1>(v);
  v += dpp<DPP_XOR_2>(v);
  return v + dpp<DPP_HALF_MIRROR>(v);
}

template <int LPT> __device__ __forceinline__ float lanes_max(float v) {
  if constexpr (LPT >= 32) {
    const TwoHalves h = halves_16(v);
    v = fmaxf(h.a, h.b);
  }
  if constexpr (LPT >= 16) v = fmaxf(v, dpp<DPP_ROTATE(8)>(v));
  v = fmaxf(v, dpp<DPP_XOR_1>(v));
  v = fmaxf(v, dpp<DPP_XOR_2>(v));
  return fmaxf(v, dpp<DPP_HALF_MIRROR>(v));
}

__device__ __forceinline__ void load4(const bf16* p, float* x) {
  const uint2 r = *reinterpret_cast<const uint2*>(p);
  x[0] = __uint_as_float(r.x << 16); x[1] = __uint_as_float(r.x & 0xffff0000u);
  x[2] = __uint_as_float(r.y << 16); x[3] = __uint_as_float(r.y & 0xffff0000u);
}
__device__ __forceinline__ void load4(const float* p, float* x) {
  const float4 r = *reinterpret_cast<const float4*>(p);
  x[0] = r.x; x[1] = r.y; x[2] = r.z; x[3] = r.w;
}

struct Append {
  const bf16* qkv;  // [T, H + 2 KV, D]
  const void* qw;   // gains [D] of the per-head norms, or null
  const void* kw;
  const float2* cs;  // [T, R / 2] cos, sin, or null
  const int* slots;  // [T]
  bf16* q_out;       // [T, H, D]
  Pages pages;
  int T, H, R;
  float eps;
  int chunk, kv_blocks;  // tokens whose runs a wave takes; workgroups of keys and values, which come first
};

// The two pieces of four coordinates of lane j of a head whose first R coordinates turn.
struct Places {
  int a, b;
  __device__ __forceinline__ Places(int j, int R) {
    const bool turns = 8 * j < R;
    a = turns ? 4 * j : 8 * j;
    b = turns ? 4 * j + R / 2 : 8 * j + 4;
  }
};

// Norm (gains g, or none) and rotation of a head's eight coordinates in this lane by the angles of token t.  busy: the lane has coordinates of its own;
// one that has none holds lane 0's, which are turned as there: largest magnitudes are taken over all lanes.
template <int D>
__device__ __forceinline__ void norm_turn(float (&x)[8], bool norm, const float (&g)[8], const float2* cs, float eps, int R, int t, int j, bool busy) {
  if (!busy) j = 0;
  const bool turns = 8 * j < R;
  float4 a, b;
  if (turns) {
    const float4* angles = reinterpret_cast<const float4*>(cs + (size_t)t * (R / 2) + 4 * j);
    a = angles[0];
    b = angles[1];
  }
  if (norm) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
    const float inv = __builtin_amdgcn_rsqf(lanes_sum<Lanes<D>::LPT>(D == 192 && !busy ? 0.f : ss) * (1.f / (float)D) + eps);  // to one step of fp32
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * g[i];
  }
  if (turns) {
    const float c[4] = {a.x, a.z, b.x, b.z}, s[4] = {a.y, a.w, b.y, b.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float u = x[i], v = x[4 + i];
      x[i] = u * c[i] - v * s[i];
      x[4 + i] = v * c[i] + u * s[i];
    }
  }
}

template <int D, typename W> __device__ __forceinline__ void append_query(const Append& a, unsigned unit, int j) {
  const int t = unit / a.H, h = unit - t * a.H;
  if (t >= a.T) return;  // whole groups leave
  const bool busy = 8 * j < D;
  const Places at(busy ? j : 0, a.R);
  const bf16* src = a.qkv + ((size_t)t * (a.H + 2 * a.pages.KV) + h) * D;
  float x[8], g[8];
  load4(src + at.a, x);
  load4(src + at.b, x + 4);
  if (a.qw) {
    load4((const W*)a.qw + at.a, g);
    load4((const W*)a.qw + at.b, g + 4);
  }
  norm_turn<D>(x, a.qw != nullptr, g, a.cs, a.eps, a.R, t, j, busy);
  if (!busy) return;
  bf16* dst = a.q_out + ((size_t)t * a.H + h) * D;
  *reinterpret_cast<bf16x4_t*>(dst + at.a) = bf16x4_t{(bf16)x[0], (bf16)x[1], (bf16)x[2], (bf16)x[3]};
  *reinterpret_cast<bf16x4_t*>(dst + at.b) = bf16x4_t{(bf16)x[4], (bf16)x[5], (bf16)x[6], (bf16)x[7]};
}

// A run of n tokens from token t on into the places from `off` on of a block.  turned: D * 16 bytes of LDS, this wave's own.
template <int D, typename W, bool VALUES>
__device__ __forceinline__ void append_run(const Append& a, int t, int n, int slot, int kvh, const float (&g)[8], uint8_t* turned) {
  constexpr int LPT = Lanes<D>::LPT, PASSES = Lanes<D>::PASSES;
  const int lane = threadIdx.x & (WAVE - 1), group = lane / LPT, j = lane % LPT, heads = a.H + 2 * a.pages.KV, bs = a.pages.nb * BLOCK;
  const bool busy = 8 * j < D;
  const int R = VALUES ? 0 : a.R, off = slot % BLOCK;
  const Places at(busy ? j : 0, R);
  const size_t block = block_index(a.pages, slot / bs, kvh, slot % bs / BLOCK);
  const bf16* src = a.qkv + ((size_t)t * heads + a.H + (VALUES ? a.pages.KV : 0) + kvh) * D;
  float* scales = VALUES ? a.pages.vs : a.pages.ks;
  uint8_t* base = (VALUES ? a.pages.v : a.pages.k) + block * (BLOCK * D);
  // All that is read is asked for before anything is waited for.  Places that are not the run's repeat one of its tokens: nothing to choose between
  // but where results are stored.
  float x[PASSES][8];
  u32x4_t held[D / 64];
  const float before = off > 0 ? scales[block] : 0.f;  // a block that begins with this run is new
  if constexpr (VALUES) {
    if (n < BLOCK) {
#pragma unroll
      for (int i = 0; i < D / 64; ++i) held[i] = reinterpret_cast<const u32x4_t*>(base)[64 * i + lane];
    }
  }
  auto nth = [&](int p) { return min(max(group * PASSES + p - off, 0), n - 1); };
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const bf16* from = src + (size_t)nth(p) * heads * D;
    load4(from + at.a, x[p]);
    load4(from + at.b, x[p] + 4);
  }
  unsigned most = 0;  // the largest magnitude's bits
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    if constexpr (!VALUES) norm_turn<D>(x[p], a.kw != nullptr, g, a.cs, a.eps, R, t + nth(p), j, busy);
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(x[p][i]) & 0x7fffffffu);
  }
  float amax = wave_max(__uint_as_float(min(most, 0x7f800000u)));
  if (amax > LARGEST * 0x1p119f) {  // uniform, and rare: numbers that are not finite are zeros, and larger ones the largest that a scale reaches
    most = 0;
#pragma unroll
    for (int p = 0; p < PASSES; ++p)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[p][i] = __builtin_amdgcn_fmed3f(finite_or_zero(x[p][i]), -LARGEST * 0x1p119f, LARGEST * 0x1p119f);
        most = max(most, __float_as_uint(x[p][i]) & 0x7fffffffu);
      }
    amax = wave_max(__uint_as_float(most));
  }
  const float scale = fmaxf(before, block_scale(amax)), inv = inverse_of(scale);
  const bool grows = before > 0.f && scale > before;
  const float by = before * inv;
  if constexpr (!VALUES) {
    if (grows) {  // the block's other rows at the new scale
      for (int w = lane; w < BLOCK * D / 4; w += WAVE) {
        const int row = 4 * w / D;
        unsigned* word = reinterpret_cast<unsigned*>(base) + w;
        if (row < off || row >= off + n) *word = rescale4(*word, by);
      }
    }
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int place = group * PASSES + p;
      if (busy && place >= off && place < off + n) {
        *reinterpret_cast<unsigned*>(base + place * D + at.a) = pack4(x[p][0] * inv, x[p][1] * inv, x[p][2] * inv, x[p][3] * inv);
        *reinterpret_cast<unsigned*>(base + place * D + at.b) = pack4(x[p][4] * inv, x[p][5] * inv, x[p][6] * inv, x[p][7] * inv);
      }
    }
  } else {
    if (busy) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint8_t* to = turned + (8 * j + i) * BLOCK + group * PASSES;
        if constexpr (PASSES == 2) {
          *reinterpret_cast<uint16_t*>(to) = (uint16_t)pack4(x[0][i] * inv, x[1][i] * inv, 0.f, 0.f);
        } else {
#pragma unroll
          for (int p = 0; p < PASSES; p += 4)
            *reinterpret_cast<unsigned*>(to + p) = pack4(x[p][i] * inv, x[p + 1][i] * inv, x[p + 2][i] * inv, x[p + 3][i] * inv);
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // a wave's own bytes: nobody else to wait for
    u32x4_t mine;  // which bytes of a coordinate's 16 are the run's
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      mine[w] = 0u;
#pragma unroll
      for (int b = 0; b < 4; ++b)
        if (4 * w + b >= off && 4 * w + b < off + n) mine[w] |= 0xffu << (8 * b);
    }
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      u32x4_t out = *reinterpret_cast<const u32x4_t*>(turned + (64 * i + lane) * BLOCK);
      if (n < BLOCK) {
        if (grows)
#pragma unroll
          for (int w = 0; w < 4; ++w) held[i][w] = rescale4(held[i][w], by);
        out = (out & mine) | (held[i] & ~mine);
      }
      reinterpret_cast<u32x4_t*>(base)[64 * i + lane] = out;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  if (lane == 0) scales[block] = scale;
}

// Single tokens (decode steps), as many as a wave has groups of lanes, each group one: `tokens` has the lanes that look at them, `slot` what lane l looks at.
// Nothing crosses lanes: a key is a row, a value a byte of every coordinate's 16, and only a scale that grows makes the rest of the block be read.
// Lane j has every (D / 8)th coordinate of a value, from j on: neighbours' bytes are 16 apart, and a store is a few lines of memory instead of one a lane.
template <int D, typename W, bool VALUES>
__device__ __forceinline__ void append_singles(const Append& a, int t0, unsigned long long& tokens, int slot, int kvh, const float (&g)[8]) {
  constexpr int LPT = Lanes<D>::LPT, AT_ONCE = Lanes<D>::AT_ONCE;
  const int lane = threadIdx.x & (WAVE - 1), group = lane / LPT, j = lane % LPT, heads = a.H + 2 * a.pages.KV, bs = a.pages.nb * BLOCK;
  const bool busy = 8 * j < D;
  const int R = VALUES ? 0 : a.R;
  const Places at(busy ? j : 0, R);
  int t = -1, s = 0;
#pragma unroll
  for (int i = 0; i < AT_ONCE; ++i) {
    if (!tokens) break;  // uniform
    const int l = __builtin_ctzll(tokens), here = __builtin_amdgcn_readlane(slot, l);
    tokens &= tokens - 1;
    if (group >= i) {  // groups beyond the last token repeat it and store nothing
      t = group == i ? t0 - 1 + l : -1;
      s = here;
    }
  }
  const bool mine = t >= 0;
  if (!mine) return;  // whole groups leave
  const int off = s % BLOCK;
  const size_t block = block_index(a.pages, s / bs, kvh, s % bs / BLOCK);
  float* scales = VALUES ? a.pages.vs : a.pages.ks;
  uint8_t* base = (VALUES ? a.pages.v : a.pages.k) + block * (BLOCK * D);
  const bf16* src = a.qkv + ((size_t)t * heads + a.H + (VALUES ? a.pages.KV : 0) + kvh) * D;
  const float before = off > 0 ? scales[block] : 0.f;  // a block that begins with this token is new
  float x[8];
  if constexpr (VALUES) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)src[D / 8 * i + (busy ? j : 0)];
  } else {
    load4(src + at.a, x);
    load4(src + at.b, x + 4);
  }
  if constexpr (!VALUES) norm_turn<D>(x, a.kw != nullptr, g, a.cs, a.eps, R, t, j, busy);
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = __builtin_amdgcn_fmed3f(finite_or_zero(x[i]), -LARGEST * 0x1p119f, LARGEST * 0x1p119f);
    amax = fmaxf(amax, fabsf(x[i]));
  }
  const float scale = fmaxf(before, block_scale(lanes_max<LPT>(amax))), inv = inverse_of(scale), by = before * inv;
  const bool grows = before > 0.f && scale > before;
  const unsigned lower = pack4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv), upper = pack4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
  if constexpr (!VALUES) {
    if (grows)  // the block's other rows at the new scale
      for (int w = j; w < BLOCK * D / 4; w += LPT) {
        unsigned* word = reinterpret_cast<unsigned*>(base) + w;
        if (4 * w / D != off) *word = rescale4(*word, by);
      }
    if (busy) {
      *reinterpret_cast<unsigned*>(base + off * D + at.a) = lower;
      *reinterpret_cast<unsigned*>(base + off * D + at.b) = upper;
    }
  } else if (busy) {
    const unsigned shift = 8 * (off & 3);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned byte = (i < 4 ? lower : upper) >> (8 * (i & 3)) & 0xffu;
      uint8_t* piece = base + (D / 8 * i + j) * BLOCK;
      if (grows) {
        u32x4_t held = *reinterpret_cast<const u32x4_t*>(piece);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          held[w] = rescale4(held[w], by);
          if (off >> 2 == w) held[w] = (held[w] & ~(0xffu << shift)) | byte << shift;
        }
        *reinterpret_cast<u32x4_t*>(piece) = held;
      } else {
        piece[off] = (uint8_t)byte;
      }
    }
  }
  if (j == 0) scales[block] = scale;
}

template <int D, typename W> __global__ __launch_bounds__(256) void append8_kernel(Append a) {
  constexpr int LPT = Lanes<D>::LPT;
  __shared__ __align__(16) uint8_t turned[4][D * BLOCK];
  const int lane = threadIdx.x & (WAVE - 1), j = lane % LPT, KV = a.pages.KV;
  if ((int)blockIdx.x >= a.kv_blocks) {
    append_query<D, W>(a, (blockIdx.x - a.kv_blocks) * (256 / LPT) + threadIdx.x / LPT, j);
    return;
  }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int id = blockIdx.x * 4 + wave, unit = id % (2 * KV), t0 = id / (2 * KV) * a.chunk;
  if (t0 >= a.T) return;
  const bool values = unit >= KV;
  const int kvh = values ? unit - KV : unit;
  // lane l looks at token t0 - 1 + l
  const int t = t0 - 1 + lane;
  const int slot = t >= 0 && t < a.T ? a.slots[t] : -2;
  const int before = __shfl(slot, max(lane - 1, 0), WAVE);
  const bool goes_on = slot > 0 && slot % BLOCK != 0 && before == slot - 1;  // in the run of the token before it
  const unsigned long long on = __ballot(goes_on);
  unsigned long long first = __ballot(lane >= 1 && lane <= a.chunk && slot >= 0 && slot / (a.pages.nb * BLOCK) < a.pages.num_pages && !goes_on);
  float g[8];
  const W* gains = (const W*)a.kw;
  if (!values && gains && first) {
    const Places at(8 * j < D ? j : 0, a.R);
    load4(gains + at.a, g);
    load4(gains + at.b, g + 4);
  }
  // first: the lanes whose tokens begin a run of this wave's; a run of one has nobody that goes on behind it
  unsigned long long singles = first & ~(on >> 1), runs = first & on >> 1;
  while (singles) {  // uniform
    if (values) append_singles<D, W, true>(a, t0, singles, slot, kvh, g);
    else append_singles<D, W, false>(a, t0, singles, slot, kvh, g);
  }
  while (runs) {
    const int l = __builtin_ctzll(runs);
    runs &= runs - 1;
    const int n = __builtin_ctzll(~(on >> (l + 1))) + 1, s = __builtin_amdgcn_readlane(slot, l);
    if (values) append_run<D, W, true>(a, t0 - 1 + l, n, s, kvh, g, turned[wave]);
    else append_run<D, W, false>(a, t0 - 1 + l, n, s, kvh, g, turned[wave]);
  }
}

// ---- attention --------------------------------------------------------------------------------------------
//
// A wave owns 16 columns, each a query of one head: the heads of a group for one token, or 16 queries of a prompt's tile.  It walks the keys in
// steps of 64, four blocks, one of them each lane group's:
//
//   S^T[key][column] = K Q^T     the e4m3 keys as they are (16x16x128, 8-bit operands).  A query is scaled by a power of two as a block is and
//                                split in two e4m3 parts, the number rounded and what is left of it: 4 + 4 bits hold a bf16 number's eight
//                                exactly, down to 2^-9.8 of the query's largest coordinate, and what is smaller is off by 2^-17.8 of it at most
//                                (half a smallest step, 2^-10, where the largest is 224 or more).  The instruction adds 32-bit sums of eight
//                                neighbouring coordinates each, but aligns those eight products first: what lies under 2^-13 of the largest one's
//                                power of two is cut off, towards zero.  So a score is off by up to 2^-10 of the largest product of every eight.
//                                Heads of even coordinates do not notice (2.1e-3 against 64 bits, as over 16 bits); a coordinate that adds 30,
//                                100, 1,000 to every score makes it 3.7e-3, 1.3e-2, 4.6e-2 (four such coordinates 2.4e-3, 4.4e-3, 1.3e-2), where
//                                keeping the keys of such heads in 8 bits has moved results by 0.7 and more, and of even ones by 2.7e-2.  bf16 keys
//                                would take as long in the matrix cores and a conversion each on the vector unit.
//   softmax                      fp32, base 2, what weights are relative to and their sums kept per column
//   O^T[d][column] += V^T P^T    values as bf16 (exact, the scale included), weights rounded to bf16: the matrix cores' operands, a part of 2^-8 at most
//
// The denominator is the 32-bit sum of the weights: as they are for single queries, rounded for portions, where the matrix cores add them up.  Either way a
// result is off by that part of the weighted magnitudes, as over 16-bit pages.
//
// Row r of score tile tt (0 .. 3) stands for key 16 (r / 4) + 4 tt + r % 4 of a step, so that the 16 keys whose weights a lane holds after the score
// product are one block: one scale, and in the transposed values 16 bytes a coordinate.
constexpr int STEP = 64;

template <int D> struct Query {
  u32x4_t high[D / 64], low[D / 64];  // coordinates 64 c + 16 grp .. + 15 of this lane's column
  float scale;
  float sum;  // what the sum of its weights begins with
  // No e4m3 numbers stand for a query that is not finite.  Its scores count as 0, so that they move no maximum, and its sum is NaN: its result
  // is, and none of its neighbours'.
  __device__ __forceinline__ void finite_or_not(float amax) {
    const bool finite = amax < __builtin_inff();
    scale = finite ? scale : 0.f;
    sum = finite ? 0.f : __builtin_nanf("");
  }
};

// Four numbers of a query, scaled, as their two parts.
__device__ __forceinline__ void split4(const float* x, float inv, unsigned& high, unsigned& low) {
  float y[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) y[n] = at_most_largest(x[n] * inv);
  high = pack4(y[0], y[1], y[2], y[3]);
  const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)high, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)high, true);
  low = pack4(y[0] - a[0], y[1] - a[1], y[2] - b[0], y[3] - b[1]);
}

template <int D> __device__ __forceinline__ void load_query(Query<D>& q, const bf16* row, int grp) {
  float x[D / 64][16];
  unsigned most = 0;  // the largest magnitude's bits: of a query that is not finite those of an infinity or more
#pragma unroll
  for (int c = 0; c < D / 64; ++c)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      load4(row + 64 * c + 16 * grp + i, x[c] + i);
#pragma unroll
      for (int n = 0; n < 4; ++n) most = max(most, __float_as_uint(x[c][i + n]) & 0x7fffffffu);
    }
  const float amax = quad_rows_max(__uint_as_float(min(most, 0x7f800000u)));
  q.scale = block_scale(amax);
  const float inv = inverse_of(q.scale);
#pragma unroll
  for (int c = 0; c < D / 64; ++c)
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      unsigned high, low;
      split4(x[c] + 4 * w, inv, high, low);
      q.high[c][w] = high;
      q.low[c][w] = low;
    }
  q.finite_or_not(amax);
}

__device__ __forceinline__ i32x8_t both(u32x4_t a, u32x4_t b) {
  return i32x8_t{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}

// scores of 16 keys, k: this lane's key, 16 bytes of every 64 coordinates
template <int D> __device__ __forceinline__ f32x4_t score_tile(const u32x4_t (&k)[D / 64], const Query<D>& q) {
  f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c + 1 < D / 64; c += 2) {
    const i32x8_t kk = both(k[c], k[c + 1]);
    s = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(kk, both(q.high[c], q.high[c + 1]), s, 0, 0, 0, 0, 0, 0);
    s = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(kk, both(q.low[c], q.low[c + 1]), s, 0, 0, 0, 0, 0, 0);
  }
  if constexpr ((D / 64) % 2) {  // 64 coordinates that are left: both parts at once
    constexpr int c = D / 64 - 1;
    s = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(both(k[c], k[c]), both(q.high[c], q.low[c]), s, 0, 0, 0, 0, 0, 0);
  }
  return s;
}

// What scores are taken relative to need not be their maximum: half of it is as good.  So the reference is SLACK (a factor of 2) above the maximum that moved it
// last, a maximum up to there moves nothing, and whether one is beyond is all that a step asks; lanes agree on a new one, and sums are rescaled, only then.  2,048
// tokens behind 14,336 take 458 us, 485 where every step does all of it, 472 where it does so for any growth and 445 where it does so for a growth beyond 2^8;
// but a largest weight that is no power of two is rounded to bfloat16 itself: errors against 64 bits are 1.93e-3, 1.88e-3, 1.88e-3 and 2.12e-3.
//
// A weight is 2^(score x factor - reference) by one fused operation, whose product is not rounded, while a maximum is a rounded product: from 2^24 on the two are
// up to SLACK apart and more, from 2^31 on a weight would be infinite, or all of them 0.  There the reference is 2 to 4 steps below the maximum instead, and weights,
// which are 1 at most anyway, are cut at 1 by the exponential's own clamp, which is free: what 32 bits hardly tell from the maximum weighs as much.
constexpr float SLACK = 1.f;  // in base 2
__device__ __forceinline__ float reference_of(float top) { return fabsf(top) < 0x1p24f ? top + SLACK : top - fabsf(top) * 0x1p-22f; }
__device__ __forceinline__ float weight_of(float score, float by, float base) {
  return __builtin_amdgcn_fmed3f(__builtin_amdgcn_exp2f(fmaf(score, by, -base)), 0.f, 1.f);
}

template <int D> struct Running {
  f32x4_t o[D / 16];
  float m, l;  // the column's reference (base 2; -inf: nothing seen), and the sum of this lane's weights
  __device__ __forceinline__ void clear(const Query<D>& q) {
#pragma unroll
    for (int d = 0; d < D / 16; ++d) o[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    m = NEG_INF;
    l = q.sum;
  }
};

// The blocks of a step's keys as a request's table names them.  Keys are uniform over the wave and its scalar unit finds them: the division by a page's
// blocks is a product with `magic` = ceil(2^32 / blocks), exact while 16-token blocks of a context times blocks of a page stay under 2^32.
// Entries that are none of the pool's (of pages given back) are read as page 0, and keys beyond the last as those of its block: numbers, which masks hide.
struct Pieces {
  const int* entries;
  int last;  // the last block that a query sees
  unsigned magic;
};
struct Blocks {  // pages as the table has them, and blocks within a page; asked for here, looked at a step later
  unsigned p0, p1, p2, p3, s0, s1, s2, s3;
  static __device__ __forceinline__ void ask(const Pages& pages, const Pieces& pieces, int key, unsigned& page, unsigned& sub) {
    const unsigned n = min(key / BLOCK, pieces.last), entry = __umulhi(n, pieces.magic) + n * (pages.nb == 1);
    page = pieces.entries[entry];
    sub = n - entry * pages.nb;
  }
  __device__ __forceinline__ void ask(const Pages& pages, const Pieces& pieces, int kb) {
    ask(pages, pieces, kb, p0, s0);
    ask(pages, pieces, kb + BLOCK, p1, s1);
    ask(pages, pieces, kb + 2 * BLOCK, p2, s2);
    ask(pages, pieces, kb + 3 * BLOCK, p3, s3);
  }
  static __device__ __forceinline__ unsigned of(const Pages& p, int kvh, unsigned page, unsigned sub) {
    return ((page < (unsigned)p.num_pages ? page : 0u) * p.KV + kvh) * p.nb + sub;
  }
};

// The operands of a step as they lie in memory.
template <int D> struct Held {
  u32x4_t k[4][D / 64];  // of score tile tt: this lane's key, 16 bytes of every 64 coordinates
  u32x4_t v[D / 16];     // the lane group's 16 keys of coordinate 16 d + col
  float ks, vs;
};

template <int D> __device__ __forceinline__ void load_step(Held<D>& held, const Pages& pages, Blocks b, int kvh) {
  const int lane = threadIdx.x & (WAVE - 1), col = lane & 15, grp = lane >> 4;
  const unsigned b0 = Blocks::of(pages, kvh, b.p0, b.s0), b1 = Blocks::of(pages, kvh, b.p1, b.s1);
  const unsigned b2 = Blocks::of(pages, kvh, b.p2, b.s2), b3 = Blocks::of(pages, kvh, b.p3, b.s3);
  const unsigned kblock = col & 8 ? (col & 4 ? b3 : b2) : (col & 4 ? b1 : b0), vblock = grp & 2 ? (grp & 1 ? b3 : b2) : (grp & 1 ? b1 : b0);
  const uint8_t* krow = pages.k + (size_t)kblock * (BLOCK * D) + (col & 3) * D + 16 * grp;
#pragma unroll
  for (int tt = 0; tt < 4; ++tt)
#pragma unroll
    for (int c = 0; c < D / 64; ++c) held.k[tt][c] = *reinterpret_cast<const u32x4_t*>(krow + 4 * tt * D + 64 * c);
  held.ks = pages.ks[vblock];
  held.vs = pages.vs[vblock];
  const uint8_t* vcol = pages.v + (size_t)vblock * (BLOCK * D) + BLOCK * col;
#pragma unroll
  for (int d = 0; d < D / 16; ++d) held.v[d] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(vcol + 16 * BLOCK * d));
}

// 16 e4m3 values (keys 0 .. 15 of a coordinate) times 2^n as bf16: exact
__device__ __forceinline__ void widen(const u32x4_t& v, float scale, bf16x8_t (&out)[2]) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * h + w], scale, false);
      const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * h + w], scale, true);
      out[h][4 * w] = a[0]; out[h][4 * w + 1] = a[1]; out[h][4 * w + 2] = b[0]; out[h][4 * w + 3] = b[1];
    }
}

__device__ __forceinline__ float max_of_16(const f32x4_t (&s)[4]) {
  const float m0 = max3(s[0][0], s[0][1], s[0][2]), m1 = max3(s[0][3], s[1][0], s[1][1]), m2 = max3(s[1][2], s[1][3], s[2][0]);
  const float m3 = max3(s[2][1], s[2][2], s[2][3]), m4 = max3(s[3][0], s[3][1], s[3][2]);
  return max3(max3(m0, m1, m2), max3(m3, m4, s[3][3]), NEG_INF);
}

// What a score of e4m3 numbers is multiplied by: the query's factor times the block's scale, 0 of a block that was never written.  Kept a normal number:
// either is as small as 2^-100 where all is zero, and a scale can be that of keys that are hidden, but a hidden score's -inf times 0, or a score of 0 times
// infinity, would be NaN.
__device__ __forceinline__ float score_unit(float factor, float scale) { return __builtin_amdgcn_fmed3f(factor * scale, 0x1p-126f, 0x1.fffffep127f); }

// A step's products and softmax for queries of one token (pos, lo uniform).  factor: from a score of e4m3 numbers to one in base 2 (to one in caps where
// scores are capped), without the block's scale.
template <int D>
__device__ __forceinline__ void take_step(const Held<D>& held, int kb, const Query<D>& q, float factor, float cap, int pos, int lo, int keep,
                                          Running<D>& run) {
  const int grp = (threadIdx.x & (WAVE - 1)) >> 4;
  f32x4_t s[4];
#pragma unroll
  for (int tt = 0; tt < 4; ++tt) s[tt] = score_tile<D>(held.k[tt], q);
  float by = score_unit(factor, held.ks);
  if (cap > 0.f) {  // uniform
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[tt][r] = quick_tanh(s[tt][r] * by);
    by = cap * LOG2E;
  }
  if (kb + STEP - 1 > pos || kb < lo) {  // uniform
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int key = kb + 16 * grp + 4 * tt + r;
        s[tt][r] = key <= pos && (key >= lo || key < keep) ? s[tt][r] : NEG_INF;
      }
  }
  const float top = max_of_16(s) * by;
  if (__any(top > run.m)) {  // uniform; rare once the first keys have been seen
    const float mn = fmaxf(run.m, reference_of(quad_rows_max(top)));
    const float alpha = __builtin_amdgcn_exp2f(run.m - (mn == NEG_INF ? 0.f : mn));
    run.m = mn;
    run.l *= alpha;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) run.o[d] *= alpha;
  }
  const float base = run.m == NEG_INF ? 0.f : run.m;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  bf16x8_t p[2];
#pragma unroll
  for (int tt = 0; tt < 4; ++tt)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float w = weight_of(s[tt][r], by, base);
      sum[r] += w;
      p[tt >> 1][(tt & 1) * 4 + r] = (bf16)w;
    }
  run.l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
  for (int d = 0; d < D / 16; ++d) {
    bf16x8_t v[2];
    widen(held.v[d], held.vs, v);
#pragma unroll
    for (int h = 0; h < 2; ++h) run.o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[h], p[h], run.o[d], 0, 0, 0);
  }
}

// Which steps of 64 keys a walk takes: those from the sequence's start that hold kept tokens, then those from the first key in sight on.
struct Steps {
  int kept, base, count;
  __device__ __forceinline__ Steps(int lo, int keep, int last) {  // lo: the first key of any column's window; last: the last key
    const int k = min(keep, lo);
    kept = (k + STEP - 1) / STEP;
    base = lo / STEP;
    if (kept > 0 && kept >= base) kept = base = 0;
    count = last < 0 ? 0 : kept + last / STEP - base + 1;
  }
  __device__ __forceinline__ int first_key(int at) const { return STEP * (at < kept ? at : at - kept + base); }
};

// Four neighbouring results, as bf16 or, with `wide`, fp32.
__device__ __forceinline__ void put4(bf16* out, size_t i, f32x4_t v, int wide) {
  if (wide) *reinterpret_cast<f32x4_t*>(reinterpret_cast<float*>(out) + i) = v;
  else *reinterpret_cast<bf16x4_t*>(out + i) = bf16x4_t{(bf16)v[0], (bf16)v[1], (bf16)v[2], (bf16)v[3]};
}

// Division by a number that a whole grid divides by, as a product: exact while dividend times divisor stays under 2^32.
struct Divide {
  unsigned by, magic;
  explicit Divide(unsigned by) : by(by), magic(by > 1 ? (unsigned)((0x100000000ull + by - 1) / by) : 0u) {}
  __device__ __forceinline__ int operator()(unsigned n) const { return by == 1 ? n : __umulhi(n, magic); }
};

struct Attend {
  const bf16* q;
  Pages pages;
  const int* items;      // single queries: the tokens, or null for all
  const int* positions;
  const int* tok_row;    // null: token t is row t
  const int* tiles;      // portions: [num_tiles, 4] first token, count, row, first position
  const int* tables;
  int table_width;
  bf16* out;
  float *part_m, *part_l, *part_acc;
  int H, KV, share;      // KV: groups of query heads; `share` of them read one head of the pages
  float scale;
  Sight sight;
  int part_steps, P;
  unsigned magic;  // of a page's blocks (`Pieces`)
  int cus;
  Divide kv, group;  // by KV and H / KV
};

__device__ __forceinline__ float score_factor(const Attend& a) { return a.scale * (a.sight.cap > 0.f ? __builtin_amdgcn_rcpf(a.sight.cap) : LOG2E); }

// The weighted sum over its denominator; nothing seen: 0.  m in base 2.
__device__ __forceinline__ float share_of(const Sight& sight, int head, float m, float l) {
  if (sight.sink) {
    const float sk = sink_score(1, sight.sinks, head) * LOG2E, top = fmaxf(m, sk), e = __builtin_amdgcn_exp2f(m - top);
    if (top == NEG_INF) return 0.f;  // a sink of no weight, beside nothing
    return e / (l * e + __builtin_amdgcn_exp2f(sk - top));
  }
  return l == 0.f ? 0.f : 1.0f / l;
}

// FRESH: the kernel takes the projection's output instead of finished queries and does what `append8_kernel` does before a decode step whose tokens are
// their own rows: a workgroup norms and turns its group's queries, the new key and value, lane group by lane group, and hands them round in LDS; the
// wave whose step ends with the token's own position puts key and value into the operands that it has just loaded and writes them to the block, whose
// scale it may raise.  Only that wave reads or writes the token's block, so nothing waits for it.  The same numbers as in two kernels, in one launch.
struct Fresh {
  Append from;  // q_out, chunk and kv_blocks are not used
  int store;    // 0: queries only, the block already holds the token
};

// A query as the lanes that normed it leave it in LDS: the parts that `load_query` makes.
template <int D> struct Split {
  unsigned high[D / 4], low[D / 4];
  float scale, amax;
  unsigned apart[2];
};

// The token's key and value as its block holds them, in LDS.
template <int D> struct News {
  unsigned bytes[2][D / 4];
  float scale[2];  // the block's, with the token
  float by[2];     // what the block's other numbers are multiplied by: below 1 where the scale grows
};

// They go into the operands of the step that holds the token, its place in the step being `nth`, and with `write` into the block.  All that LDS holds is read at
// once and chosen from without branches: reading where it was needed, this took 1.4 us of a wave that everybody waits for.
template <int D>
__device__ __forceinline__ void insert(Held<D>& held, const News<D>& news, int nth, const Pages& pages, unsigned block, bool write) {
  const int lane = threadIdx.x & (WAVE - 1), col = lane & 15, grp = lane >> 4, piece = nth >> 4, off = nth & 15;
  u32x4_t key[D / 64];
  unsigned value[D / 16];
#pragma unroll
  for (int c = 0; c < D / 64; ++c) key[c] = *reinterpret_cast<const u32x4_t*>(&news.bytes[0][16 * c + 4 * grp]);
#pragma unroll
  for (int d = 0; d < D / 16; ++d) value[d] = news.bytes[1][4 * d + (col >> 2)];
  const float kby = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(news.by[0])));
  const float vby = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(news.by[1])));
  const float ks = news.scale[0], vs = news.scale[1];
  const bool my_keys = col >> 2 == piece, my_values = grp == piece;  // this lane's are the block's
  uint8_t* const rows = pages.k + (size_t)block * (BLOCK * D) + 16 * grp;
  if (kby < 1.f && my_keys) {
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
#pragma unroll
        for (int w = 0; w < 4; ++w) held.k[tt][c][w] = rescale4(held.k[tt][c][w], kby);
        if (write) *reinterpret_cast<u32x4_t*>(rows + (4 * tt + (col & 3)) * D + 64 * c) = held.k[tt][c];
      }
  }
#pragma unroll
  for (int tt = 0; tt < 4; ++tt) {
    const bool hit = my_keys && 4 * tt + (col & 3) == off;
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
#pragma unroll
      for (int w = 0; w < 4; ++w) held.k[tt][c][w] = hit ? key[c][w] : held.k[tt][c][w];
  }
  if (write && my_keys && (col & 3) == (off & 3)) {
#pragma unroll
    for (int c = 0; c < D / 64; ++c) *reinterpret_cast<u32x4_t*>(rows + off * D + 64 * c) = key[c];
  }
  if (vby < 1.f && my_values) {
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
#pragma unroll
      for (int w = 0; w < 4; ++w) held.v[d][w] = rescale4(held.v[d][w], vby);
  }
  const unsigned byte = my_values ? 0xffu << (8 * (off & 3)) : 0u;
  unsigned mine[4];  // where the value's byte lies in a coordinate's 16
#pragma unroll
  for (int w = 0; w < 4; ++w) mine[w] = off >> 2 == w ? byte : 0u;
  u32x4_t* const vcol = reinterpret_cast<u32x4_t*>(pages.v + (size_t)block * (BLOCK * D)) + col;
#pragma unroll
  for (int d = 0; d < D / 16; ++d) {
    const unsigned fresh = (value[d] >> (8 * (col & 3)) & 0xffu) << (8 * (off & 3));
#pragma unroll
    for (int w = 0; w < 4; ++w) held.v[d][w] = (held.v[d][w] & ~mine[w]) | (fresh & mine[w]);
  }
  held.ks = my_values ? ks : held.ks;
  held.vs = my_values ? vs : held.vs;
  if (write && my_values) {
#pragma unroll
    for (int d = 0; d < D / 16; ++d) vcol[16 * d] = held.v[d];
    if (col == 0) {
      pages.ks[block] = ks;
      pages.vs[block] = vs;
    }
  }
}

// One workgroup per (token, group of query heads, partition of its keys); its four waves take the steps in turn.  W: of FRESH, the gains' type.
//
// Bound by the pages' bytes as soon as there are enough of them: 64 contexts of 300 to 8,000 tokens (32 heads of 128 on 8) 80 to 82 us, 6.6 TB/s (a large
// copy reads and writes 5.1); one of 131,005 (64 heads on 8) 45 us with its merge, 5.9 TB/s.  16-bit pages: 183 and 84.  A step's operands go from memory into
// registers in the order in which the matrix instructions take them: LDS would hold the same bytes once more, and nobody shares them, since all heads of a
// group are columns of one wave.  Two steps in flight a wave (one being taken, one on its way) hide most of the latency: the
// form that loaded a step when it came to it took 252 us for the 64 contexts.
// Where there is little to read, latency is the bound: 700 keys of one request 6.5 us (16-bit pages 6.6), of which a launch, the page's entry, the
// operands and the exchange between waves wait for one another.
template <int D, bool FRESH, typename W>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void single8_kernel(Attend a, Fresh fresh) {
  constexpr int LD = D + 4;
  extern __shared__ __align__(16) float smem[];  // [4][16] m, [4][16] l, [4][G][LD]; FRESH: the news, [G] queries
  const int G = a.group.by, part = blockIdx.y;
  int item = a.kv(blockIdx.x), kvh = blockIdx.x - item * a.KV;
  if (a.P == 1 && (int)gridDim.x > a.cus) {
    // Whole contexts of unequal length, a workgroup each, two of them on a compute unit.  Taken eight items at a time, their kv heads one after the
    // other, with the second round of workgroups backwards: with `items` sorted longest first a compute unit's first two are a long and a short one.
    int s = blockIdx.x;
    const int total = gridDim.x, N = a.kv(total);
    if (s >= a.cus && s < 2 * a.cus) s = a.cus + (min(2 * a.cus, total) - 1 - s);
    const int first = s / (8 * a.KV) * 8, r = s % (8 * a.KV), here = min(8, N - first);
    item = first + r % here;
    kvh = r / here;
  }
  const int h0 = kvh * G;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, grp = lane >> 4;
  const int t = a.items ? a.items[item] : item, bs = a.pages.nb * BLOCK;
  const int* const table = a.tables + (size_t)(a.tok_row ? a.tok_row[t] : t) * a.table_width;
  const int from = part * a.part_steps;
  int at = from + wave;
  // Where nothing hides the first keys, the entries of the first step are asked for beside the position: those beyond it, whatever they are, name
  // numbers that the mask hides.
  const bool whole = a.sight.window == 0 && a.sight.chunk == 0;
  Blocks blocks{};
  if (whole) blocks.ask(a.pages, Pieces{table, a.table_width * a.pages.nb - 1, a.magic}, STEP * min(at, (a.table_width * a.pages.nb - 1) / (STEP / BLOCK)));
  const int pos = min(a.positions[t], a.table_width * bs - 1);
  const int lo = first_in_window(a.sight, pos + 1);
  const Pieces pieces{table, max(pos, 0) / BLOCK, a.magic};
  const Steps steps(lo, a.sight.keep, pos);
  const int to = min(steps.count, from + a.part_steps);
  [[maybe_unused]] const int last = steps.count - 1;  // the step that ends with the token's own position
  [[maybe_unused]] const bool here = FRESH && fresh.store && last >= from && last < to;
  [[maybe_unused]] unsigned own_block = 0;
  [[maybe_unused]] bool write = false;  // whether the token is kept
  if constexpr (FRESH) {
    if (here) {
      Blocks own;
      own.ask(a.pages, pieces, pos);
      const int slot = fresh.from.slots[t];
      own_block = Blocks::of(a.pages, kvh, own.p0, own.s0);
      write = slot >= 0 && slot / bs < a.pages.num_pages && block_index(a.pages, slot / bs, kvh, slot % bs / BLOCK) == own_block;
    }
  }
  // a step's operands are asked for a step ahead, where they lie two steps ahead
  Held<D> even, odd;
  const int page_head = a.share > 1 ? kvh / a.share : kvh;
  if (at < to) {
    if (!whole) blocks.ask(a.pages, pieces, steps.first_key(at));
    load_step<D>(even, a.pages, blocks, page_head);
    if (at + 4 < to) blocks.ask(a.pages, pieces, steps.first_key(at + 4));
  }
  Query<D> q;
  [[maybe_unused]] News<D>* const news = reinterpret_cast<News<D>*>(smem + 128 + 4 * LD * G);
  if constexpr (FRESH) {
    constexpr int LPT = Lanes<D>::LPT, AT_ONCE = Lanes<D>::AT_ONCE;
    const Append& f = fresh.from;
    Split<D>* const queries = reinterpret_cast<Split<D>*>(news + 1);
    const int j = lane % LPT, jobs = G + (here ? 2 : 0), heads = a.H + 2 * a.KV;
    const bool busy = 8 * j < D;
    for (int job = wave * AT_ONCE + lane / LPT; job < jobs; job += 4 * AT_ONCE) {  // the group's queries, the key, the value; whole lane groups
      const bool query = job < G, key = job == G;
      const Places at8(busy ? j : 0, job <= G ? f.R : 0);
      const bf16* src = f.qkv + ((size_t)t * heads + (query ? h0 + job : a.H + kvh + (key ? 0 : a.KV))) * D;
      float x[8], g[8], before = 0.f;
      load4(src + at8.a, x);
      load4(src + at8.b, x + 4);
      if (!query && pos % BLOCK > 0) before = (key ? a.pages.ks : a.pages.vs)[own_block];  // a block that begins with this token is new
      const W* gains = (const W*)(query ? f.qw : f.kw);
      if (gains) {
        load4(gains + at8.a, g);
        load4(gains + at8.b, g + 4);
      }
      if (job <= G) norm_turn<D>(x, gains != nullptr, g, f.cs, f.eps, f.R, t, j, busy);
      if (query) {
        unsigned most = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = (float)(bf16)x[i];
          most = max(most, __float_as_uint(x[i]) & 0x7fffffffu);
        }
        const float amax = lanes_max<LPT>(busy ? __uint_as_float(min(most, 0x7f800000u)) : 0.f), scale = block_scale(amax), inv = inverse_of(scale);
        if (!busy) continue;
        Split<D>& to8 = queries[job];
        split4(x, inv, to8.high[at8.a / 4], to8.low[at8.a / 4]);
        split4(x + 4, inv, to8.high[at8.b / 4], to8.low[at8.b / 4]);
        if (j == 0) {
          to8.scale = scale;
          to8.amax = amax;
        }
      } else {
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = __builtin_amdgcn_fmed3f(finite_or_zero(x[i]), -LARGEST * 0x1p119f, LARGEST * 0x1p119f);
          amax = fmaxf(amax, fabsf(x[i]));
        }
        const float scale = fmaxf(before, block_scale(lanes_max<LPT>(amax))), inv = inverse_of(scale);
        const int which = key ? 0 : 1;
        if (busy) {
          news->bytes[which][at8.a / 4] = pack4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
          news->bytes[which][at8.b / 4] = pack4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
        }
        if (j == 0) {
          news->scale[which] = scale;
          news->by[which] = before > 0.f ? before * inv : 1.f;
        }
      }
    }
    __syncthreads();
    const Split<D>& from8 = queries[min(col, G - 1)];
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      q.high[c] = *reinterpret_cast<const u32x4_t*>(&from8.high[16 * c + 4 * grp]);
      q.low[c] = *reinterpret_cast<const u32x4_t*>(&from8.low[16 * c + 4 * grp]);
    }
    q.scale = from8.scale;
    q.finite_or_not(from8.amax);
  } else {
    load_query<D>(q, a.q + ((size_t)t * a.H + h0 + min(col, G - 1)) * D, grp);
  }
  const float factor = score_factor(a) * q.scale;
  Running<D> run;
  run.clear(q);
  auto turn = [&](Held<D>& now, Held<D>& next) {
    if constexpr (FRESH) {
      if (here && at == last) {  // uniform: this wave's step holds the token itself
        insert<D>(now, *news, pos % STEP, a.pages, own_block, write);
      }
    }
    if (at + 4 < to) {
      load_step<D>(next, a.pages, blocks, page_head);
      if (at + 8 < to) blocks.ask(a.pages, pieces, steps.first_key(at + 8));
    }
    take_step<D>(now, steps.first_key(at), q, factor, a.sight.cap, pos, lo, a.sight.keep, run);
    at += 4;
  };
  while (at < to) {
    turn(even, odd);
    if (at < to) turn(odd, even);
  }
  run.l = quad_rows_sum(run.l);
  float *sm = smem, *sl = smem + 64, *so = smem + 128;
  if (grp == 0 && col < G) { sm[wave * 16 + col] = run.m; sl[wave * 16 + col] = run.m == NEG_INF ? 0.f : run.l; }
  if (col < G)
#pragma unroll
    for (int d = 0; d < D / 16; ++d) *reinterpret_cast<f32x4_t*>(so + (wave * G + col) * LD + d * 16 + 4 * grp) = run.o[d];
  __syncthreads();
  for (int i = tid; i < G * D / 4; i += 256) {  // four coordinates a thread
    const int g = i / (D / 4), d = i % (D / 4) * 4, h = h0 + g;
    float m = NEG_INF, den = 0.f, ms[4], ls[4];
    f32x4_t num = {0.f, 0.f, 0.f, 0.f}, acc[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      ms[w] = sm[w * 16 + g];
      ls[w] = sl[w * 16 + g];
      acc[w] = *reinterpret_cast<const f32x4_t*>(so + (w * G + g) * LD + d);
      m = fmaxf(m, ms[w]);
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float e = m == NEG_INF ? 0.f : __builtin_amdgcn_exp2f(ms[w] - m);
      num += acc[w] * e;
      den += ls[w] * e;
    }
    if (a.P == 1) {
      put4(a.out, ((size_t)t * a.H + h) * D + d, num * share_of(a.sight, h, m, den), a.sight.wide);
    } else {
      const size_t o = ((size_t)item * a.H + h) * a.P + part;
      *reinterpret_cast<f32x4_t*>(a.part_acc + o * D + d) = num;
      if (d == 0) { a.part_m[o] = m; a.part_l[o] = den; }
    }
  }
}

// The partitions of every (token, head): sum acc_p 2^(m_p - m) / sum l_p 2^(m_p - m).  A lane holds a partition's weight and hands it round by lane
// reads; maxima, sums and the first eight outputs are asked for at once, and nothing waits for another.  A thread has a coordinate (D is whole waves).
__global__ __launch_bounds__(256) void single8_merge_kernel(Attend a, int D) {
  const int item = blockIdx.x, h = blockIdx.y, t = a.items ? a.items[item] : item, lane = threadIdx.x & (WAVE - 1), d = threadIdx.x;
  const size_t base = ((size_t)item * a.H + h) * a.P;
  const float* acc = a.part_acc + base * D + d;
  float v[8];
  auto ask = [&](int p) {  // eight at a time; those past the end repeat the last with a weight of 0
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = acc[(size_t)min(p + j, a.P - 1) * D];
  };
  ask(0);
  float mp = lane < a.P ? a.part_m[base + lane] : NEG_INF, lp = lane < a.P ? a.part_l[base + lane] : 0.f, m = mp;
  for (int p = lane + WAVE; p < a.P; p += WAVE) m = fmaxf(m, a.part_m[base + p]);
  m = wave_max(m);
  float num = 0.f, den = 0.f;
  for (int p0 = 0; p0 < a.P; p0 += WAVE) {
    if (p0 > 0) {
      mp = p0 + lane < a.P ? a.part_m[base + p0 + lane] : NEG_INF;
      lp = p0 + lane < a.P ? a.part_l[base + p0 + lane] : 0.f;
    }
    const float weight = mp == NEG_INF ? 0.f : __builtin_amdgcn_exp2f(mp - m), l = weight == 0.f ? 0.f : lp * weight;
    const int here = min(WAVE, a.P - p0);
    for (int p = 0; p < here; p += 8) {
      if (p0 + p > 0) ask(p0 + p);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        den += __int_as_float(__builtin_amdgcn_readlane(__float_as_int(l), p + j));
        num = fmaf(v[j], __int_as_float(__builtin_amdgcn_readlane(__float_as_int(weight), p + j)), num);
      }
    }
  }
  put(a.out, ((size_t)t * a.H + h) * D + d, num * share_of(a.sight, h, m, den), a.sight.wide);
}

// ---- portions of prompts ------------------------------------------------------------------------------------
//
// Work item: up to 64 consecutive tokens of one request for one kv head and four waves of queries.  A wave owns 16 QT queries of one head as QT column
// tiles; the waves of a workgroup take heads of one group or other queries of the tile, so that all need the same keys and values.  Those come into LDS
// a round of 64 keys ahead, a wave one block of four:
//
//   keys     as they are, by copies that pass no register (buffer_load ... lds).  16-byte piece c of key k lies at c ^ swizzle(k): the 16 rows of a
//            score tile, keys 4 tt .. + 3 of four blocks, lie in different banks.
//   values   through registers, widened to bf16 on the way (once a workgroup instead of once a wave: the vector unit has the softmax to do):
//            slot (2 block + h) D + d holds keys 8 h .. + 7 of coordinate d, so that 16 lanes read 256 bytes in one piece.
//
// One barrier a round.  Where the blocks lie and their scales are looked up for 16 rounds at a time, a block a lane.
//
// Bound by the matrix cores' products and the softmax between them, at the clock that is left: with QT 2 and heads of 128 a wave's round is 52 products (1,090
// cycles); matrix cores are busy 57 per cent of the time and the vector unit 49.  Sums of weights are products with ones, which the vector unit would take 128
// cycles for (2 to 4 per cent of the time).  2,048 tokens behind 14,336 (32 heads on 8): 442 to 467 us, 1,104 to 1,166 TFLOP/s where an 8192^3
// bf16 product reaches 1,212; 16-bit pages 535.  Keys read by every wave from memory, without LDS, took 1,561.  A ring of four rounds in LDS was
// 3 to 20 per cent slower (room for fewer workgroups), a round's weighted values under the next round's softmax 15 (spills), widening between
// the weighted values' products and wave priorities no different.
//
// A step of few work items takes as long as its longest one: with `pieces` > 1 an item comes as that many workgroups, an item of more than `piece_rounds`
// rounds is cut along its keys, and what the pieces leave (maxima, sums, unnormalised outputs) is put together by a second kernel.
struct Cut {
  int pieces, piece_rounds;
  int* cut;    // [items]: the pieces of each (1: not cut)
  float* ml;   // [T, H, pieces, 2] what weights are relative to (base 2), sum
  float* acc;  // [T, H, pieces, D]
};

template <int D> __device__ __forceinline__ int swizzle(int key) {  // of a key within a round
  const int block = key >> 4 & 3;
  return D == 256 ? (key & 3) | block << 2 : D == 128 ? (key >> 1 & 1) | block << 1 : block;
}

struct Item {  // what a workgroup and a wave of it work on
  int item, tile, kvh, bz, piece;
  __device__ __forceinline__ Item(const Attend& a, const Divide& units_z, const Divide& pass, const Divide& pieces) {
    // Items in the order of `tiles`, those that see most keys first; runs of `pass` of them alternate direction, so that a compute unit that
    // received one of the longest in one round of workgroups receives one of the shortest in the next.
    int n = blockIdx.x;
    const int block = pass(n), first = block * pass.by, size = min((int)pass.by, (int)gridDim.x - first);
    if (block & 1) n = first + size - 1 - (n - first);
    item = pieces(n);
    piece = n - item * pieces.by;
    split(a, units_z);
  }
  __device__ __forceinline__ Item(const Attend& a, const Divide& units_z, int item) : item(item) { split(a, units_z); }
  __device__ __forceinline__ void split(const Attend& a, const Divide& units_z) {
    const int heads = units_z(item);
    bz = item - heads * units_z.by;
    tile = a.kv(heads);
    kvh = heads - tile * a.KV;
  }
};

template <int D, int QT>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void prompt8_kernel(Attend a, Divide units_z, Divide pass, Divide pieces, Cut cut) {
  constexpr int DT = D / 16, WQ = 16 * QT, PARTS = 64 / WQ;  // queries of a wave; waves that share a head's 64 queries
  constexpr int KEYS = STEP * D, VALUES = 2 * STEP * D;      // bytes of a round
  __shared__ __align__(128) char keys[2][KEYS];
  __shared__ __align__(128) char values[2][VALUES];
  const Item it(a, units_z, pass, pieces);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, grp = lane >> 4;
  const int G = a.group.by, kvh = it.kvh, end = a.table_width * a.pages.nb * BLOCK - 1;
  const int tok0 = a.tiles[4 * it.tile], count = a.tiles[4 * it.tile + 1], pos0 = max(a.tiles[4 * it.tile + 3], 0);
  const int* const table = a.tables + (size_t)a.tiles[4 * it.tile + 2] * a.table_width;
  auto first_seen = [&](int pos) { return first_in_window(a.sight, pos + 1); };

  // the keys this workgroup walks: from the first key that any of its waves sees to the last
  int wg_lo = 0x7fffffff, wg_last = -1;
  for (int u = it.bz * 4; u < it.bz * 4 + 4 && u < PARTS * G; ++u) {
    const int uq0 = a.group(u) * WQ;
    if (uq0 >= count) continue;
    wg_last = max(wg_last, min(pos0 + min(count, uq0 + WQ) - 1, end));
    wg_lo = min(wg_lo, first_seen(min(pos0 + uq0, end)));
  }
  if (wg_last < 0) {  // uniform over the workgroup
    if (cut.pieces > 1 && it.piece == 0 && tid == 0) cut.cut[it.item] = 1;
    return;
  }
  const int keep = a.sight.keep;
  const Steps steps(wg_lo, keep, wg_last);
  int rd_first = 0, rd_end = steps.count;
  bool partial = false;  // this workgroup leaves its share of a cut item for the merge
  if (cut.pieces > 1) {
    const int mine = min(cut.pieces, (rd_end + cut.piece_rounds - 1) / cut.piece_rounds);
    if (it.piece == 0 && tid == 0) cut.cut[it.item] = mine;
    if (it.piece >= mine) return;
    if (mine > 1) {
      partial = true;
      rd_first = cut.piece_rounds * it.piece;
      if (it.piece + 1 < mine) rd_end = rd_first + cut.piece_rounds;
    }
  }
  const int rounds = rd_end - rd_first;

  // this wave's queries
  const int unit = it.bz * 4 + wave, part = a.group(unit), head = kvh * G + unit - part * G, q0 = part * WQ;
  const bool working = unit < PARTS * G && q0 < count;
  const int nq = working ? min(WQ, count - q0) : 1;
  const int my_first = min(pos0 + q0, end), my_last = working ? min(pos0 + q0 + nq - 1, end) : -1;
  const int my_lo = first_seen(my_first), last_lo = first_seen(my_last);
  Query<D> q[QT];
  Running<D> run[QT];
  int qpos[QT], qlo[QT];
  float factor[QT];
  float base[QT];  // the columns' references; 0 while there is none
  f32x4_t l[QT];  // sums of weights, the same in every row: the weights' product with ones
  bf16x8_t ones;
#pragma unroll
  for (int i = 0; i < 8; ++i) ones[i] = (bf16)1.f;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    base[qt] = 0.f;
    const int qc = min(qt * 16 + col, nq - 1);  // columns past the end repeat the last query and are not stored
    qpos[qt] = min(pos0 + q0 + qc, end);
    qlo[qt] = first_seen(qpos[qt]);
    load_query<D>(q[qt], a.q + ((size_t)(tok0 + (working ? q0 + qc : 0)) * a.H + head) * D, grp);
    factor[qt] = score_factor(a) * q[qt].scale;
    run[qt].clear(q[qt]);
    l[qt] = f32x4_t{run[qt].l, run[qt].l, run[qt].l, run[qt].l};
  }

  // where blocks lie: lane l has block l % 4 of round 16 batch + l / 4
  const int last_block = wg_last / BLOCK;
  auto place_of = [&](int batch) {
    const int rd = min(16 * batch + (lane >> 2), rounds - 1);
    return min(steps.first_key(rd_first + rd) / BLOCK + (lane & 3), last_block);
  };
  auto entry_of = [&](int n) { return a.pages.nb == 1 ? n : (int)__umulhi(n, a.magic); };
  int page_ahead = table[entry_of(place_of(0))];
  unsigned block = 0;
  float ks_ahead = 0.f, vs_ahead = 0.f;
  auto locate = [&](int batch) {
    const int n = place_of(batch);
    const unsigned page = (unsigned)page_ahead < (unsigned)a.pages.num_pages ? page_ahead : 0u;
    block = (page * a.pages.KV + kvh) * a.pages.nb + (n - entry_of(n) * a.pages.nb);
    ks_ahead = a.pages.ks[block];
    vs_ahead = a.pages.vs[block];
    page_ahead = table[entry_of(place_of(batch + 1))];
  };

  // this wave's share of a round: block `wave` of four
  int k_at[D / 64];  // the byte of a block that this lane copies
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    const int slot = 64 * i + lane, key = slot / (D / 16), c = slot % (D / 16);
    k_at[i] = key * D + (c ^ swizzle<D>(16 * wave + key)) * 16;
  }
  u32x4_t raw[D / 64];  // values on their way
  size_t at = 0;
  auto aim = [&](int rd) {
    if ((rd & 15) == 0) locate(rd >> 4);
    at = (size_t)(unsigned)__builtin_amdgcn_readlane(block, 4 * (rd & 15) + wave) * (BLOCK * D);
  };
  auto copy_keys = [&](int rd) {
    const __amdgpu_buffer_rsrc_t buf = __builtin_amdgcn_make_buffer_rsrc(a.pages.k + at, 0, BLOCK * D, 0x00020000);
    const unsigned to = (unsigned)(uintptr_t)(wide::lds_char*)&keys[rd & 1][wave * BLOCK * D];
#pragma unroll
    for (int i = 0; i < D / 64; ++i) wide::copy_to_lds(buf, k_at[i], 0u, to + 1024 * i);
  };
  auto ask_values = [&]() {
    const u32x4_t* from = reinterpret_cast<const u32x4_t*>(a.pages.v + at) + lane;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) raw[i] = from[64 * i];
  };
  auto put_values = [&](int rd) {  // the block's scale is the wave's own: lane 4 r + wave of the batch
    const float scale = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs_ahead), 4 * (rd & 15) + wave));
    u32x4_t* const to = reinterpret_cast<u32x4_t*>(values[rd & 1]) + 2 * wave * D + lane;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      bf16x8_t v[2];
      widen(raw[i], scale, v);
      to[64 * i] = __builtin_bit_cast(u32x4_t, v[0]);
      to[64 * i + D] = __builtin_bit_cast(u32x4_t, v[1]);
    }
  };
  const int swz = swizzle<D>(16 * (col >> 2) + (col & 3));
  const char* const krow = keys[0] + (16 * (col >> 2) + (col & 3)) * D;

  float ks_now = 0.f;
  aim(0);
  copy_keys(0);
  ask_values();
  put_values(0);
  for (int rd = 0; rd < rounds; ++rd) {
    if ((rd & 15) == 0) ks_now = ks_ahead;  // the batch that this round belongs to, before the copies' next one
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const bool more = rd + 1 < rounds;
    if (more) {
      aim(rd + 1);
      copy_keys(rd + 1);
      ask_values();
    }
    const int kb = steps.first_key(rd_first + rd);
    if (working && kb <= my_last && (kb + STEP - 1 >= my_lo || kb < keep)) {  // uniform over the wave
      const float ks = __shfl(ks_now, 4 * (rd & 15) + grp, WAVE);
      f32x4_t s[QT][4];
      u32x4_t k[2][D / 64];
      auto read_keys = [&](int tt, u32x4_t (&into)[D / 64]) {
#pragma unroll
        for (int c = 0; c < D / 64; ++c) into[c] = *reinterpret_cast<const u32x4_t*>(krow + (rd & 1) * KEYS + 4 * tt * D + ((4 * c + grp) ^ swz) * 16);
      };
      read_keys(0, k[0]);
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        if (tt < 3) read_keys(tt + 1, k[(tt + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);  // or the compiler moves every read down to its product
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) s[qt][tt] = score_tile<D>(k[tt & 1], q[qt]);
      }
      u32x4_t v[2][DT];
      auto read_values = [&](int h) {
        const u32x4_t* from = reinterpret_cast<const u32x4_t*>(values[rd & 1]) + (2 * grp + h) * D + col;
#pragma unroll
        for (int d = 0; d < DT; ++d) v[h][d] = from[16 * d];
      };
      constexpr bool EARLY = D <= 128;  // asked for before the softmax, as far as registers hold them
      if constexpr (EARLY) read_values(0);
      __builtin_amdgcn_sched_barrier(0);
      const bool masked = kb + STEP - 1 > my_first || kb < last_lo;
      bf16x8_t p[QT][2];
      float by[QT], top[QT];  // top: the largest score of this lane's 16
      bool grows = false;
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        by[qt] = score_unit(factor[qt], ks);
        if (a.sight.cap > 0.f) {
#pragma unroll
          for (int tt = 0; tt < 4; ++tt)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[qt][tt][r] = quick_tanh(s[qt][tt][r] * by[qt]);
          by[qt] = a.sight.cap * LOG2E;
        }
        if (masked) {
#pragma unroll
          for (int tt = 0; tt < 4; ++tt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int key = kb + 16 * grp + 4 * tt + r;
              s[qt][tt][r] = key <= qpos[qt] && (key >= qlo[qt] || key < keep) ? s[qt][tt][r] : NEG_INF;
            }
        }
        top[qt] = max_of_16(s[qt]) * by[qt];
        grows = grows || top[qt] > run[qt].m;
      }
      if (__any(grows)) {  // uniform; rare once the first keys have been seen
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          const float mn = fmaxf(run[qt].m, reference_of(quad_rows_max(top[qt])));
          base[qt] = mn == NEG_INF ? 0.f : mn;
          const float alpha = __builtin_amdgcn_exp2f(run[qt].m - base[qt]);
          run[qt].m = mn;
          l[qt] *= alpha;
#pragma unroll
          for (int d = 0; d < DT; ++d) run[qt].o[d] *= alpha;
        }
      }
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
          for (int r = 0; r < 4; ++r) p[qt][tt >> 1][(tt & 1) * 4 + r] = (bf16)weight_of(s[qt][tt][r], by[qt], base[qt]);
      if constexpr (!EARLY) read_values(0);
      read_values(1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) l[qt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, p[qt][h], l[qt], 0, 0, 0);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int qt = 0; qt < QT; ++qt)
            run[qt].o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, v[h][d]), p[qt][h], run[qt].o[d], 0, 0, 0);
    }
    if (more) put_values(rd + 1);
  }

#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    if (!working || qt * 16 + col >= nq) continue;
    const size_t row = (size_t)(tok0 + q0 + qt * 16 + col) * a.H + head;
    if (partial) {
      const size_t to = row * cut.pieces + it.piece;
      if (grp == 0) *reinterpret_cast<float2*>(cut.ml + 2 * to) = make_float2(run[qt].m, l[qt][0]);
#pragma unroll
      for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4_t*>(cut.acc + to * D + 16 * d + 4 * grp) = run[qt].o[d];
      continue;
    }
    const float inv = share_of(a.sight, head, run[qt].m, l[qt][0]);
#pragma unroll
    for (int d = 0; d < DT; ++d) put4(a.out, row * D + 16 * d + 4 * grp, run[qt].o[d] * inv, a.sight.wide);
  }
}

// The pieces of every cut item, put together: out = sum_j acc_j 2^(m_j - m) / sum_j l_j 2^(m_j - m).  A workgroup per item and 32 coordinates, lanes as
// above.  Two, four or eight pieces are asked for at once, before their maxima are known: one piece after the other is a chain of as many waits (64 tokens
// behind 8,000, 32 heads, 8 pieces: attention and merge 35.6 us with that chain, now 28.7).
template <int D, int AT_ONCE>
__device__ __forceinline__ void merge_row(const Attend& a, const Cut& cut, size_t row, int head, int n, int at) {
  const size_t from = row * cut.pieces;
  float m = NEG_INF, den = 0.f;
  f32x4_t sum[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  for (int j0 = 0; j0 < n; j0 += AT_ONCE) {
    float2 ml[AT_ONCE];
    f32x4_t acc[AT_ONCE][2];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {  // those past the last repeat it, with a weight of 0
      const size_t piece = from + min(j0 + j, n - 1);
      ml[j] = reinterpret_cast<const float2*>(cut.ml)[piece];
#pragma unroll
      for (int d = 0; d < 2; ++d) acc[j][d] = *reinterpret_cast<const f32x4_t*>(cut.acc + piece * D + at + 16 * d);
    }
    float top = m;
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) top = fmaxf(top, ml[j].x);
    const float base = top == NEG_INF ? 0.f : top, past = __builtin_amdgcn_exp2f(m - base);
    den *= past;
#pragma unroll
    for (int d = 0; d < 2; ++d) sum[d] *= past;
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const float w = j0 + j < n ? __builtin_amdgcn_exp2f(ml[j].x - base) : 0.f;
      den += ml[j].y * w;
#pragma unroll
      for (int d = 0; d < 2; ++d) sum[d] += acc[j][d] * w;
    }
    m = top;
  }
  const float inv = share_of(a.sight, head, m, den);
#pragma unroll
  for (int d = 0; d < 2; ++d) put4(a.out, row * D + at + 16 * d, sum[d] * inv, a.sight.wide);
}

template <int D, int QT>
__global__ __launch_bounds__(256) void prompt8_merge_kernel(Attend a, Divide units_z, Cut cut) {
  constexpr int WQ = 16 * QT, PARTS = 64 / WQ;
  const int item = blockIdx.x, n = cut.cut[item];
  if (n <= 1) return;
  const Item it(a, units_z, item);
  const int G = a.group.by, tile = it.tile;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, at = 32 * blockIdx.y + 4 * (lane >> 4);
  const int tok0 = a.tiles[4 * tile], count = a.tiles[4 * tile + 1];
  const int unit = it.bz * 4 + wave, part = a.group(unit), head = it.kvh * G + unit - part * G, q0 = part * WQ;
  if (unit >= PARTS * G || q0 >= count) return;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int qi = q0 + qt * 16 + col;
    if (qi >= count) continue;
    const size_t row = (size_t)(tok0 + qi) * a.H + head;
    if (n <= 2) merge_row<D, 2>(a, cut, row, head, n, at);
    else if (n <= 4) merge_row<D, 4>(a, cut, row, head, n, at);
    else merge_row<D, 8>(a, cut, row, head, n, at);
  }
}

template <typename... T> bool on_16_bytes(const T*... p) { return !(((uintptr_t)p | ...) & 15); }
bool pages_ok(const void* k, const void* v, const float* ks, const float* vs, int num_pages, int KV, int D, int bs) {
  return k && v && ks && vs && num_pages > 0 && KV > 0 && D > 0 && D % 64 == 0 && D <= 256 && bs > 0 && bs % BLOCK == 0 &&
         on_16_bytes(k, v);
}
// ceil(2^32 / blocks of a page); a page of one block needs none
unsigned magic_of(int bs) { return bs > BLOCK ? (unsigned)((0x100000000ull + bs / BLOCK - 1) / (bs / BLOCK)) : 0u; }
bool table_ok(int num_pages, int KV, int bs, int table_width) {  // block numbers fit 32 bits, and their division by a page's is exact
  const long long nb = bs / BLOCK;
  return table_width > 0 && (long long)num_pages * KV * nb <= 0xffffffffll && table_width * nb <= 0x7ffffffll && table_width * nb * nb <= 0xffffffffll;
}
Pages pages_of(const void* k, const void* v, const float* ks, const float* vs, int num_pages, int KV, int bs) {
  return Pages{(uint8_t*)k, (uint8_t*)v, (float*)ks, (float*)vs, num_pages, KV, bs / BLOCK};
}

}  // namespace

#define FOR_WIDTH(CALL)       \
  switch (D / 64) {           \
    case 1: CALL(64); break;  \
    case 2: CALL(128); break; \
    case 3: CALL(192); break; \
    default: CALL(256); break; \
  }

// Per-head norm (qw, kw: gains [D], or null), rotation of the first R coordinates in pairs (i, i + R/2) (cs [T, R/2] cos, sin, or null),
// queries to q_out [T, H, D] and, with store, keys and values into the blocks that `slots` name (page * bs + offset; none for a negative one).
// qkv [T, H + 2 KV, D] bf16; D a multiple of 64 up to 256, R of 8, bs of 16.  Tokens of one block come as one run: next to each other, in the
// order of their places; a run that starts at a block's first place makes it new.
extern "C" int as_qk_norm_rope_store8(const void* qkv, const void* qw, const void* kw, int w_dtype, const float* cs, const int* slots,
                                      void* q_out, void* k_pages, void* v_pages, float* k_scales, float* v_scales, int num_pages, int num_tokens,
                                      int H, int KV, int D, int R, float eps, int bs, int store, hipStream_t stream) {
  if (num_tokens <= 0) return AS_OK;
  if (H <= 0 || KV <= 0 || D <= 0 || D % 64 || D > 256 || R < 0 || R > D || R % 8 || (R > 0) != (cs != nullptr)) return AS_BAD_SHAPE;
  if ((qw == nullptr) != (kw == nullptr) || !qkv || !q_out || !on_16_bytes(qkv, qw, kw, cs, q_out)) return AS_BAD_SHAPE;
  if (store && (!slots || !pages_ok(k_pages, v_pages, k_scales, v_scales, num_pages, KV, D, bs))) return AS_BAD_SHAPE;
  if (w_dtype != DT_F32 && w_dtype != DT_BF16) return AS_BAD_DTYPE;
  if (R == 0) cs = nullptr;
  // Tokens whose runs a wave takes: 16 is a block, so that a prompt's waves have one run each, but single tokens, four at a time, are a chain of up to four
  // turns then.  us with 4 / 8 / 16, 32 heads of 128 on 8: single tokens of 64 requests 4.0 / 4.9 / 6.8, of 256 4.8 / 5.7 / 7.4, of 512 6.7 / 6.5 / 8.1; prompts
  // of 512 5.4 / 5.0 / 4.9, of 2,048 17.5 / 14.0 / 11.8, of 480 beside 32 single tokens 5.5 / 5.2 / 7.0.  Other widths and
  // numbers of kv heads go by the same number of (token, kv head) pairs and were not swept.
  const long long pairs = (long long)num_tokens * KV;
  const int chunk = pairs <= 2048 ? 4 : pairs <= 6144 ? 8 : 16;
  const long long kv_blocks = store ? (((long long)num_tokens + chunk - 1) / chunk * 2 * KV + 3) / 4 : 0;
  const Append a{(const bf16*)qkv, qw, kw, (const float2*)cs, slots, (bf16*)q_out, pages_of(k_pages, v_pages, k_scales, v_scales, num_pages, KV, bs),
           num_tokens, H, R, eps, chunk, (int)kv_blocks};
#define LAUNCH(DV)                                                                                       \
  {                                                                                                      \
    constexpr int groups = 256 / Lanes<DV>::LPT;                                                         \
    const long long blocks = kv_blocks + ((long long)num_tokens * H + groups - 1) / groups;              \
    if (blocks * groups > 0x7fffffffll) return AS_BAD_SHAPE;                                             \
    if (w_dtype == DT_F32) append8_kernel<DV, float><<<(int)blocks, 256, 0, stream>>>(a);                \
    else append8_kernel<DV, bf16><<<(int)blocks, 256, 0, stream>>>(a);                                   \
  }
  FOR_WIDTH(LAUNCH)
#undef LAUNCH
  return launch_status();
}

// Single queries.  parts: fp32 [N, H, P, D + 2] where P > 1, unnormalised outputs, then maxima, then sums; part_size: keys of a partition, a multiple of 64; share: how
// many of the KV groups of query heads (at most 16 to a group) read one head of the pages, which hold KV / share.
extern "C" int as_attn_single_query8(const void* q, const void* k_pages, const void* v_pages, const float* k_scales, const float* v_scales,
                                     int num_pages, const int* items, int num_items, const int* positions, const int* tok_row,
                                     const int* block_tables, int table_width, void* out, float* parts, int H,
                                     int KV, int D, int bs, float scale, int window, int keep, int chunk, float cap, int sink,
                                     const float* sinks, int wide, int part_size, int P, int share, hipStream_t stream) {
  if (num_items <= 0) return AS_OK;
  const Sight sight{window, keep, chunk, cap, sink, sinks, wide};
  if (!sight_ok(sight) || H <= 0 || KV <= 0 || H % KV || H / KV > 16 || share < 1 || KV % share) return AS_BAD_SHAPE;
  if (!pages_ok(k_pages, v_pages, k_scales, v_scales, num_pages, KV / share, D, bs) || !table_ok(num_pages, KV / share, bs, table_width)) return AS_BAD_SHAPE;
  if (!q || !positions || !block_tables || !out || !on_16_bytes(q, out, parts) || part_size <= 0 || part_size % STEP || P <= 0 || P > 65535 || (long long)num_items * KV * KV > 0xffffffffll)
    return AS_BAD_SHAPE;
  if (P > 1 && !parts) return AS_BAD_SHAPE;
  const size_t rows = P > 1 ? (size_t)num_items * H * P : 0;
  const Attend a{(const bf16*)q, pages_of(k_pages, v_pages, k_scales, v_scales, num_pages, KV / share, bs), items, positions, tok_row, nullptr,
                 block_tables, table_width, (bf16*)out, parts + rows * D, parts + rows * (D + 1), parts, H, KV, share, scale, sight, part_size / STEP, P,
                 magic_of(bs), compute_units(), Divide(KV), Divide(H / KV)};
  const size_t shmem = sizeof(float) * (128 + 4 * (size_t)(D + 4) * (H / KV));
#define LAUNCH(DV)                                                                                                                       \
  {                                                                                                                                      \
    const auto kernel = single8_kernel<DV, false, bf16>;                                                                                 \
    if (shmem > 65536 && hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)shmem) != hipSuccess) \
      return AS_LAUNCH_FAILED;                                                                                                           \
    kernel<<<dim3(KV * num_items, P), 256, shmem, stream>>>(a, Fresh{});                                                                 \
  }
  FOR_WIDTH(LAUNCH)
#undef LAUNCH
  if (hipGetLastError() != hipSuccess) return AS_LAUNCH_FAILED;
  if (P > 1) single8_merge_kernel<<<dim3(num_items, H), D, 0, stream>>>(a, D);
  return launch_status();
}

// A decode step (token t is row t of the block tables, slots[t] the place of its own position there, or negative: attended, not kept) from the projection's
// output qkv [T, H + 2 KV, D]: append and attention in one kernel.  items [T]: the order in which tokens are taken, or null; store 0: queries only.  At most 16
// query heads of at most 192 to a kv head; window as everywhere; parts and part_size as for single queries.
extern "C" int as_attn_decode_fresh8(const void* qkv, const void* qw, const void* kw, int w_dtype, const float* cs, const int* slots, float eps,
                                     int store, void* k_pages, void* v_pages, float* k_scales, float* v_scales, int num_pages, const int* items,
                                     int num_tokens, const int* positions, const int* block_tables, int table_width, void* out, float* parts,
                                     int H, int KV, int D, int R, int bs, float scale, int window, int part_size, int P, hipStream_t stream) {
  if (num_tokens <= 0) return AS_OK;
  const Sight sight{window, 0, 0, 0.f, 0, nullptr, 0};
  if (!sight_ok(sight) || H <= 0 || KV <= 0 || H % KV || H / KV > 16 || D > 192 || R < 0 || R > D || R % 8 || (R > 0) != (cs != nullptr)) return AS_BAD_SHAPE;
  if (!pages_ok(k_pages, v_pages, k_scales, v_scales, num_pages, KV, D, bs) || !table_ok(num_pages, KV, bs, table_width)) return AS_BAD_SHAPE;
  if (!qkv || (qw == nullptr) != (kw == nullptr) || (store && !slots) || !positions || !block_tables || !out || !on_16_bytes(qkv, qw, kw, cs, out, parts))
    return AS_BAD_SHAPE;
  if (part_size <= 0 || part_size % STEP || P <= 0 || P > 65535 || (long long)num_tokens * KV * KV > 0xffffffffll) return AS_BAD_SHAPE;
  if (P > 1 && !parts) return AS_BAD_SHAPE;
  if (w_dtype != DT_F32 && w_dtype != DT_BF16) return AS_BAD_DTYPE;
  const size_t rows = P > 1 ? (size_t)num_tokens * H * P : 0;
  const Pages pages = pages_of(k_pages, v_pages, k_scales, v_scales, num_pages, KV, bs);
  const Attend a{nullptr, pages, items, positions, nullptr, nullptr, block_tables, table_width, (bf16*)out, parts + rows * D, parts + rows * (D + 1),
                 parts, H, KV, 1, scale, sight, part_size / STEP, P, magic_of(bs), compute_units(), Divide(KV), Divide(H / KV)};
  const Fresh fresh{Append{(const bf16*)qkv, qw, kw, (const float2*)cs, slots, nullptr, pages, num_tokens, H, R, eps, 0, 0}, store};
  const size_t shmem = sizeof(float) * (128 + 4 * (size_t)(D + 4) * (H / KV) + 4) + 2 * (size_t)D + (2 * (size_t)D + 16) * (H / KV);
#define LAUNCH2(DV, W)                                                                                                                   \
  {                                                                                                                                      \
    const auto kernel = single8_kernel<DV, true, W>;                                                                                     \
    if (shmem > 65536 && hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)shmem) != hipSuccess) \
      return AS_LAUNCH_FAILED;                                                                                                           \
    kernel<<<dim3(KV * num_tokens, P), 256, shmem, stream>>>(a, fresh);                                                                  \
  }
#define LAUNCH(DV) if (w_dtype == DT_F32) LAUNCH2(DV, float) else LAUNCH2(DV, bf16)
  switch (D / 64) {
    case 1: LAUNCH(64) break;
    case 2: LAUNCH(128) break;
    default: LAUNCH(192) break;
  }
#undef LAUNCH
#undef LAUNCH2
  if (hipGetLastError() != hipSuccess) return AS_LAUNCH_FAILED;
  if (P > 1) single8_merge_kernel<<<dim3(num_tokens, H), D, 0, stream>>>(a, D);
  return launch_status();
}

// Portions of prompts: tiles [num_tiles, 4] int32 (first token, count <= 64, row of block_tables, position of the first), best those that see most keys
// first.  query_tiles: 2, a wave owns 32 queries of a head; 1, 16 (twice the workgroups).  pieces > 1: items of more than piece_rounds rounds of 64 keys
// are cut; parts: 32-bit words, [T, H, pieces, D] unnormalised outputs, [T, H, pieces, 2] maxima and sums and [num_tiles * KV * ceil(64 / (16 query_tiles) *
// (H / KV) / 4)] integers, with T (`tokens`) one more than the largest token of a tile; piece_rounds * pieces covers the longest item.  pieces <= 1: none is
// cut, parts may be null.
extern "C" int as_attn_prefill8(const void* q, const void* k_pages, const void* v_pages, const float* k_scales, const float* v_scales,
                                int num_pages, const int* tiles, int num_tiles, const int* block_tables, int table_width, void* out, int H,
                                int KV, int D, int bs, float scale, int window, int keep, int chunk, float cap, int sink, const float* sinks,
                                int wide, int query_tiles, int pieces, int piece_rounds, float* parts, int tokens, hipStream_t stream) {
  if (num_tiles <= 0) return AS_OK;
  const Sight sight{window, keep, chunk, cap, sink, sinks, wide};
  if (!sight_ok(sight) || H <= 0 || KV <= 0 || H % KV || (query_tiles != 1 && query_tiles != 2)) return AS_BAD_SHAPE;
  if (!pages_ok(k_pages, v_pages, k_scales, v_scales, num_pages, KV, D, bs) || !table_ok(num_pages, KV, bs, table_width)) return AS_BAD_SHAPE;
  if (!q || !tiles || !block_tables || !out || !on_16_bytes(q, out, parts)) return AS_BAD_SHAPE;
  if (pieces < 1) pieces = 1;
  if (pieces > 1 && (piece_rounds < 1 || !parts || tokens <= 0)) return AS_BAD_SHAPE;
  const int units_z = (64 / (16 * query_tiles) * (H / KV) + 3) / 4;
  const long long items = (long long)num_tiles * KV * units_z;
  if (items * pieces > 0xffffffffll / std::max(std::max(pieces, compute_units()), std::max(units_z, KV))) return AS_BAD_SHAPE;  // `Divide`
  const Divide z(units_z), pass(compute_units()), by_pieces(pieces);
  const Attend a{(const bf16*)q, pages_of(k_pages, v_pages, k_scales, v_scales, num_pages, KV, bs), nullptr, nullptr, nullptr, tiles, block_tables,
                 table_width, (bf16*)out, nullptr, nullptr, nullptr, H, KV, 1, scale, sight, 0, 1, magic_of(bs), compute_units(), Divide(KV), Divide(H / KV)};
  const size_t rows = pieces > 1 ? (size_t)tokens * H * pieces : 0;
  const Cut how{pieces, piece_rounds, (int*)(parts + rows * (D + 2)), parts + rows * D, parts};
#define LAUNCH2(DV, QTV)                                                                                           \
  {                                                                                                                \
    prompt8_kernel<DV, QTV><<<(int)(items * pieces), 256, 0, stream>>>(a, z, pass, by_pieces, how);                \
    if (pieces > 1) prompt8_merge_kernel<DV, QTV><<<dim3((int)items, DV / 32), 256, 0, stream>>>(a, z, how);       \
  }
#define LAUNCH(DV) if (query_tiles == 1) LAUNCH2(DV, 1) else LAUNCH2(DV, 2)
  FOR_WIDTH(LAUNCH)
#undef LAUNCH
#undef LAUNCH2
  return launch_status();
}
