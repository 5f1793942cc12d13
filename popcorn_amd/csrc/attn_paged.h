// Attention of new tokens over a paged cache, grouped-query, on gfx950 matrix
// cores: o = softmax(q k^T scale) v for the last n tokens of each sequence over
// the L keys the cache holds of it (the new ones among them), token t of n seeing
// keys up to L - n + t when causal. Rows of a kv head are its group's q heads of
// every new token, token by token; rows are taken 16 at a time.
//
// Working on transposes puts one row per lane column, as in the forward of whole
// sequences (attn_fwd.hip), on the 16-row products: with g = lane / 16, n = lane % 16,
//   S^T (16 keys x 16 rows)  = K . Q^T    lane: keys 4g .. 4g + 3 of row n
//   O^T (dims x 16 rows)    += V^T . P^T  lane: keys 4g .. + 3 and 16 + 4g .. + 3 of
//                                         row n in the 32 keys of one product
// so P leaves the accumulators as the B operand as it is, with the keys of the
// product in the order that V^T is given in too. Nothing goes through LDS: a lane
// loads whole 16-byte pieces of K rows (its A operand), and of the eight V rows of
// its key group the dims VL n .. VL n + VL - 1 (VL = DL / 16); the product for dim
// e of each VL takes element e of the eight rows, packed by byte permutes. O^T then
// holds dims 4 VL g .. of row n, contiguous, in a lane.
//
// Softmax: the running maximum of a row moves only when a score exceeds it by more
// than 8 (in powers of two), which a ballot finds, so almost every step has no lane
// exchange and no rescaling; P is at most 2^8.
//
// Pages: a tile of 16 keys lies in one page. A wave looks up the pages of 64 tiles
// at once (one per lane) and reads each tile through a buffer resource based at the
// tile and ending with its last visible key, so that what lies behind a sequence's
// keys, whatever it holds, reads as zeros.
//
// Work: blocks are (row tile, chunk of keys, kv head). The chunk length is found on
// the device from the lengths, by every wave alone: about `target` chunks in all, no
// shorter than `min_chunk` keys. Sequences of more than one chunk leave partial sums
// and a second kernel joins them in order. So the launch shape depends on nothing
// that the host would have to read back, and a captured graph may be replayed with
// other lengths.
//
// Bound by HBM where a sequence has few rows: 64 sequences of 200 to 8192 keys, 32/8 heads
// of 128, bf16: 118 us, 4.8 TB/s; two of 125000, fp16: 188 us, 5.7 TB/s; 48 of 1000 to
// 32768 in MXFP4: 141 us, 4.2 TB/s beside the decoding. One of 500 keys is all latency,
// 9 us. fp32 products bound a few rows in fp32 (12 sequences of 5 tokens: 20 us).
#pragma once

#include <math.h>

#include <type_traits>

#include "api.h"
#include "attn_common.h"
#include "common.h"
#include "mxfp4.h"

namespace pk {
namespace paged {

using attn::bf16x8;
using attn::f16x8;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
// Buffer offset of dims past head_dim: past every range (each below 2^31)
constexpr int kPad = (int)0x80000000u;
constexpr float kLag = 8.f;  // how far scores may exceed the running maximum, log2

struct Args {
  const void* q;
  void* o;
  const void* k;  // cache rows, or their codes
  const void* v;
  const uint8_t* ks;  // scales of a 4-bit cache
  const uint8_t* vs;
  const int* table;  // [seqs, width]
  const int* lens;   // [seqs]
  const int* cu;     // [seqs + 1], or NULL: one token a sequence
  int64_t qt, qh;     // q strides, elements
  int64_t page, head;  // page and head strides of both caches, bytes
  int token;           // token stride
  int64_t spage, shead;  // scales: page and head strides, bytes
  int sblock;            // block stride
  int64_t table_stride;
  int width, pages, tiles_per_page;
  int elem;  // bytes of a cached value (rows)
  int tpp_shift, group_shift;  // log2 of tiles_per_page and group, or -1
  int seqs, total, heads, kv_heads, group, d;
  int causal;
  float c;        // |scale| * log2(e), at least 1e-30
  uint32_t flip;  // 0x80008000 where the scale is negative, for pairs of 16-bit q
  int split;       // whether sequences may be split
  int min_chunk;   // keys
  float target, at_once;  // blocks that run at once: a kv head's share, and all
  int items;       // blocks a kv head, and row tiles: what the workspace has room for, and offsets
  int tiles;       // that do not rise may ask for more
  // partial sums: part [items][kv_heads][rows][d], ml [items][kv_heads][rows][2], meta [1 + 4 * row tiles]
  float* part;
  float* ml;
  int* meta;
  int rows;  // rows of a block's tile that partial sums have room for
};

// Inclusive sums over a wave's lanes: within rows of 16 lanes, then rows onto the rows behind.
template <typename V> __device__ __forceinline__ V scan(V v) {
  const auto moved = [](V x, auto ctrl, auto rows) {
    return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value,
                                                             decltype(rows)::value, 0xF, false));
  };
  typedef std::integral_constant<int, 0xF> All;
  v += moved(v, std::integral_constant<int, 0x111>(), All());  // the lane 1, 2, 4 and 8 in front, in the row
  v += moved(v, std::integral_constant<int, 0x112>(), All());
  v += moved(v, std::integral_constant<int, 0x114>(), All());
  v += moved(v, std::integral_constant<int, 0x118>(), All());
  v += moved(v, std::integral_constant<int, 0x142>(), std::integral_constant<int, 0xA>());  // last lane of rows 0, 2 onto 1, 3
  v += moved(v, std::integral_constant<int, 0x143>(), std::integral_constant<int, 0xC>());  // lane 31 onto rows 2 and 3
  return v;
}

struct Seq {
  int start, n, len;
};

__device__ __forceinline__ Seq seq_of(const Args& a, int i) {
  Seq s = {i, 1, min(max(a.lens[i], 0), a.width * a.tiles_per_page * 16)};  // at most 2^30
  if (a.cu) {
    s.start = min(max(a.cu[i], 0), a.total);
    s.n = min(max(a.cu[i + 1], s.start), a.total) - s.start;
  }
  return s;
}

// Token and head in the group of a row.
__device__ __forceinline__ int token_of(const Args& a, int row) {
  return a.group_shift >= 0 ? row >> a.group_shift : row / a.group;
}

// Output of a row of a sequence that starts at token `start`.
template <typename T> __device__ __forceinline__ T* row_of(const Args& a, int start, int h, int row) {
  const int token = token_of(a, row);
  return static_cast<T*>(a.o) + ((int64_t)(start + token) * a.heads + h * a.group + row - token * a.group) * a.d;
}

struct Item {
  Seq s;
  int seq, tile, chunk, splits;
  int keys;        // of a chunk
  int tiles_base;  // row tiles in front of this sequence's
  int all_tiles;
};

// Keys of a chunk, from the sum of row tiles times keys: an even share of the blocks that
// run at once where that cuts the sequences into no more blocks than those, or none of
// them, else a third of it, so that blocks of different lengths fill each other's gaps. 48
// sequences of 1000 to 32768 keys in 4 bits, 8 heads: 159 us at an even share, 142 at half,
// 137 at a third, 153 at a sixth; two of 131071 keys: 189, 198, 201 at the first three. 128
// of 1024 keys, which an even share leaves whole: 74.6 us cut, 45.4 whole (bf16 rows 118.9,
// 104.8). A block of 4-bit keys starts in the time of many of them, so a third is at least
// 2048 there: 48 of 4096 keys 58.8 -> 51.5. A sequence's chunks are as equal as steps allow:
// 128 of 4096 keys 162 -> 135.
constexpr int kParts = 3;

template <int ROWS> __device__ __forceinline__ int chunk_of(const Args& a, float work, int tiles) {
  // 1.02: a fp32 sum of up to 2^18 terms a lane is off by less, and the room for partial sums counts on it
  const float even = fminf(work * 1.02f / a.target, 1e9f);
  const int keys = max(((int)even + 64) / 64 * 64, a.min_chunk);
  const float per = 1.f / (float)keys;
  float blocks = 0.f;
  for (int i = threadIdx.x & 63; i < a.seqs; i += 64) {
    const Seq s = seq_of(a, i);
    blocks += (float)(((unsigned)s.n * (unsigned)a.group + ROWS - 1) / ROWS) * fmaxf(ceilf((float)s.len * per), 1.f);
  }
  blocks = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, scan(blocks)), 63));
  return __builtin_amdgcn_readfirstlane(
      blocks * a.kv_heads <= a.at_once || blocks == (float)tiles ? keys
                                                                 : max(((int)(even / kParts) + 64) / 64 * 64, a.ks ? 2048 : 512));
}

// Which piece of work block x is, the same in every lane; seq < 0: none. Each wave
// finds it alone, 64 sequences at a time: the lane of a sequence counts its blocks.
template <int ROWS> __device__ __forceinline__ Item find(const Args& a, int x) {
  const int lane = threadIdx.x & 63;
  Item it;
  it.seq = -1;
  it.keys = 1 << 30;
  int tiles = 0;
  Seq s = {0, 0, 0};
  if (a.split) {
    float work = 0.f;
    for (int i = lane; i < a.seqs; i += 64) {
      s = seq_of(a, i);
      const int rt = (int)(((unsigned)s.n * (unsigned)a.group + ROWS - 1) / ROWS);
      work += (float)rt * (float)s.len;
      tiles += rt;
    }
    work = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, scan(work)), 63));
    tiles = __builtin_amdgcn_readlane(scan(tiles), 63);
    it.keys = chunk_of<ROWS>(a, work, tiles);
  }
  it.all_tiles = tiles;
  int before = 0, tiles_before = 0;
  for (int base = 0; base < a.seqs; base += 64) {
    const int i = base + lane;
    if (a.seqs > 64 || !a.split) {
      s = Seq{0, 0, 0};
      if (i < a.seqs) s = seq_of(a, i);
    }
    const int rt = (int)(((unsigned)s.n * (unsigned)a.group + ROWS - 1) / ROWS);
    const int splits = a.split ? max(1, (int)(((unsigned)s.len + (unsigned)it.keys - 1) / (unsigned)it.keys)) : 1;
    const int mine = rt * splits;
    const int upto = scan(mine), rts = scan(rt);
    const int rel = x - before;
    const uint64_t found = __ballot(rel >= upto - mine && rel < upto);
    if (found != 0) {
      const int at = __builtin_ctzll(found);
      it.seq = base + at;
      it.s.start = __builtin_amdgcn_readlane(s.start, at);
      it.s.n = __builtin_amdgcn_readlane(s.n, at);
      it.s.len = __builtin_amdgcn_readlane(s.len, at);
      it.splits = __builtin_amdgcn_readlane(splits, at);
      if (it.splits > 1) {  // as equal as a block's steps allow
        const unsigned unit = ROWS > 16 ? 32 : (a.ks ? 512 : 128);
        const unsigned share = ((unsigned)it.s.len + (unsigned)it.splits - 1) / (unsigned)it.splits;
        it.keys = min(it.keys, (int)((share + unit - 1) / unit * unit));
      }
      const int k = rel - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(mine, at));
      const int tile = it.splits == 1 ? k : (int)((unsigned)k / (unsigned)it.splits);
      it.chunk = k - tile * it.splits;
      // the last row tiles see the most keys when causal: they go first
      it.tile = __builtin_amdgcn_readlane(rt, at) - 1 - tile;
      it.tiles_base = tiles_before + __builtin_amdgcn_readlane(rts, at) - __builtin_amdgcn_readlane(rt, at);
      return it;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
    tiles_before += __builtin_amdgcn_readlane(rts, 63);
  }
  return it;
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_of(const void* base, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, bytes, 0x00020000);
}
typedef unsigned w2 __attribute__((ext_vector_type(2)));
typedef unsigned w4 __attribute__((ext_vector_type(4)));

// The tiles of 16 keys of 64 / TILES steps, a lane each: where a tile's rows lie in the
// cache (k and v alike) and how many bytes from there hold visible ones.
struct Look {
  uint64_t at, scales;  // byte offsets from the kv head's first row and scale
  int bytes;            // 0: a page that is not there, or behind the last key
  uint64_t whole, there;  // lanes whose tile has 16 visible keys, and any page
};

// key: of this lane's tile; k1: the end of the visible ones, at least 1. Every lane looks,
// those behind the last key where it lies, and selects: in a branch that only some lanes
// take, the compiler (ROCm 7.2) moved other values to other registers in front of its end,
// while it still left the rest out, and theirs were lost.
template <bool MX> __device__ __forceinline__ Look look_up(const Args& a, int seq, int64_t key, int k1) {
  Look l;
  const int tile = (int)(min(key, (int64_t)(k1 - 1)) >> 4);
  const int slot = a.tpp_shift >= 0 ? tile >> a.tpp_shift : tile / a.tiles_per_page;
  const int p = a.table[seq * a.table_stride + slot];
  const bool in = key < k1 && p >= 0 && p < a.pages;
  const int page = in ? p : 0, row = (tile - slot * a.tiles_per_page) * 16;
  const int rows = in ? (int)min(k1 - key, (int64_t)16) : 0;
  l.at = (uint64_t)page * a.page + (uint64_t)row * (unsigned)a.token;
  l.bytes = in ? (rows - 1) * a.token + (MX ? a.d / 2 : a.d * (int)a.elem) : 0;
  l.scales = MX ? (uint64_t)page * a.spage + row : 0;
  l.whole = __ballot(rows == 16);
  l.there = __ballot(rows > 0);
  return l;
}

__device__ __forceinline__ uint64_t lane64(uint64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)v, lane), hi = __builtin_amdgcn_readlane((uint32_t)(v >> 32), lane);
  return ((uint64_t)hi << 32) | lo;
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const char* base, uint64_t at, int bytes, int lane) {
  return rsrc_of(base + lane64(at, lane), __builtin_amdgcn_readlane(bytes, lane));
}

// A operand of eight 16-bit values from element e of eight rows, and of those with ones in m
template <int VW> __device__ __forceinline__ w4 pick(const uint32_t (&v)[8][VW], int e, const uint32_t (&m)[8]) {
  w4 r;
#pragma unroll
  for (int w = 0; w < 4; ++w)
    r[w] = __builtin_amdgcn_perm(v[2 * w + 1][e / 2] & m[2 * w + 1], v[2 * w][e / 2] & m[2 * w],
                                 (e & 1) ? 0x07060302u : 0x05040100u);
  return r;
}
template <int VW> __device__ __forceinline__ w4 pick(const uint32_t (&v)[8][VW], int e) {
  w4 r;
#pragma unroll
  for (int w = 0; w < 4; ++w)
    r[w] = __builtin_amdgcn_perm(v[2 * w + 1][e / 2], v[2 * w][e / 2], (e & 1) ? 0x07060302u : 0x05040100u);
  return r;
}

template <typename T> struct Mma16;
template <> struct Mma16<bf16> {
  static __device__ __forceinline__ f32x4 run(w4 a, w4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <> struct Mma16<f16> {
  static __device__ __forceinline__ f32x4 run(w4 a, w4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};

typedef float f32x2 __attribute__((ext_vector_type(2)));
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef T pair __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, pair));
}
template <typename T> __device__ __forceinline__ f32x2 unpack2(uint32_t w) {
  if constexpr (__is_same(T, bf16)) return {__builtin_bit_cast(float, w << 16), __builtin_bit_cast(float, w & 0xffff0000u)};
  typedef T pair __attribute__((ext_vector_type(2)));
  const pair p = __builtin_bit_cast(pair, w);
  return {to_f32(p.x), to_f32(p.y)};
}

// The eight values x as TERMS operands of type T whose sum they are: rounded, then
// what the rounding cut off, rounded, ...
template <typename T, int TERMS> __device__ __forceinline__ void terms_of(float (&x)[8], w4 (&out)[TERMS]) {
#pragma unroll
  for (int t = 0; t < TERMS; ++t) {
#pragma unroll
    for (int w = 0; w < 4; ++w) out[t][w] = pack2<T>(x[2 * w], x[2 * w + 1]);
    if (t + 1 < TERMS) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const f32x2 r = unpack2<T>(out[t][w]);
        x[2 * w] -= r.x, x[2 * w + 1] -= r.y;
      }
    }
  }
}

// An Inf or NaN among 16-bit values, two to a word
template <typename T> __device__ __forceinline__ bool wild2(uint32_t w) {
  const uint32_t m = sizeof(T) == 2 && __is_same(T, bf16) ? 0x7f80u : 0x7c00u;
  return (w & m) == m || ((w >> 16) & m) == m;
}

// ---------------------------------------------------------------- caches
//
// A cache reads 32 SUB keys a step into a Buf and makes products of it:
//   score  S^T of tile t                           (f32x4 of the lane's four keys)
//   pv     O^T += V^T P^T of tiles 2 u and 2 u + 1  (32 keys)
//   pv_apart  the same with every key's part added to the rows that see it alone
//   wild   whether their values hold an Inf or a NaN
// kTerms: P is the sum of two terms there and values may be an Inf.

// Key 0 .. 31 of a product of 32 is row 4 (key / 16) + key % 4 of lane group (key % 16) / 4:
// all ones there, in the lanes of that group, and zeros for the other rows.
__device__ __forceinline__ void row_masks(int key, uint32_t (&m)[8]) {
  const bool mine = (int)((threadIdx.x & 63) >> 4) == (key & 15) >> 2;
  const int row = 4 * (key >> 4) + (key & 3);
#pragma unroll
  for (int i = 0; i < 8; ++i) m[i] = mine && i == row ? 0xffffffffu : 0u;
}

// P of that key alone
template <typename W> __device__ __forceinline__ W only(const W& p, const uint32_t (&m)[8]) {
  W r;
#pragma unroll
  for (int w = 0; w < 4; ++w) r[w] = p[w] & ((m[2 * w] & 0xffffu) | (m[2 * w + 1] & 0xffff0000u));
  return r;
}

__device__ __forceinline__ void add_if(bool in, const f32x4& x, f32x4& acc) {
#pragma unroll
  for (int c = 0; c < 4; ++c) acc[c] += in ? x[c] : 0.f;
}

// Rows of 16-bit values, of q's type. P is two terms of it: one would add as much error
// as rounding the output does, and the products are not what bounds a few rows.
template <typename T_, int DL_> struct Rows16 {
  typedef T_ T;
  static constexpr int DL = DL_, VL = DL / 16, SUB = 1, QN = DL / 32, VH = VL > 8 ? 2 : 1;
  static constexpr bool kMx = false, kTerms = true;
  struct Buf {
    w4 k[2][QN];
    uint32_t v[8][VL / 2];
  };
  typedef w4 Query[QN];
  typedef w4 Prob[2];  // P of 32 keys
  const char *kb, *vb;
  int koff[QN], voff[4][VH];

  __device__ __forceinline__ void init(const Args& a, int h) {
    const int lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
    kb = static_cast<const char*>(a.k) + h * a.head;
    vb = static_cast<const char*>(a.v) + h * a.head;
#pragma unroll
    for (int j = 0; j < QN; ++j) koff[j] = 32 * j + 8 * g < a.d ? n * a.token + (32 * j + 8 * g) * 2 : kPad;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int h = 0; h < VH; ++h)
        voff[i][h] = VL * n + 8 * h < a.d ? (4 * g + i) * a.token + (VL * n + 8 * h) * 2 : kPad;
  }
  static __device__ __forceinline__ void query(const Args& a, const T* row, bool live, Query& q) {
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int j = 0; j < QN; ++j) {
      q[j] = w4{0, 0, 0, 0};
      if (live && 32 * j + 8 * g < a.d) q[j] = *reinterpret_cast<const w4*>(row + 32 * j + 8 * g) ^ a.flip;
    }
  }
  __device__ __forceinline__ void load_k(const Look& l, int at, Buf& b) const {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const auto kr = tile_rsrc(kb, l.at, l.bytes, at + u);
#pragma unroll
      for (int j = 0; j < QN; ++j) b.k[u][j] = __builtin_amdgcn_raw_buffer_load_b128(kr, koff[j], 0, 0);
    }
  }
  __device__ __forceinline__ void load_v(const Look& l, int at, Buf& b) const {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const auto vr = tile_rsrc(vb, l.at, l.bytes, at + u);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t(&to)[VL / 2] = b.v[4 * u + i];
        if constexpr (VL == 4) {
          const w2 x = __builtin_amdgcn_raw_buffer_load_b64(vr, voff[i][0], 0, 0);
          to[0] = x.x, to[1] = x.y;
        } else {
#pragma unroll
          for (int hh = 0; hh < VH; ++hh) {
            const w4 x = __builtin_amdgcn_raw_buffer_load_b128(vr, voff[i][hh], 0, 0);
#pragma unroll
            for (int w = 0; w < 4; ++w) to[4 * hh + w] = x[w];
          }
        }
      }
    }
  }
  // behind a sequence's last key everything reads as zero already
  static __device__ __forceinline__ void trim(Buf&, int) {}
  static __device__ __forceinline__ f32x4 score(const Buf& b, int t, const Query& q) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < QN; ++j) s = Mma16<T>::run(b.k[t][j], q[j], s);
    return s;
  }
  static __device__ __forceinline__ void prob(const f32x4& lo, const f32x4& hi, Prob& p) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = lo[i], x[4 + i] = hi[i];
    terms_of<T, 2>(x, p);
  }
  template <int R>
  static __device__ __forceinline__ void pv(const Buf& b, int, const Prob (&p)[R], f32x4 (&acc)[R][VL]) {
#pragma unroll
    for (int e = 0; e < VL; ++e) {
      const w4 f = pick(b.v, e);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int m = 0; m < 2; ++m) acc[r][e] = Mma16<T>::run(f, p[r][m], acc[r][e]);
    }
  }
  // The same product one key at a time, added to the rows that see it: in(r, key). P's first
  // term alone: an Inf times it and times a second one, 0 or of the other sign, is a NaN.
  template <int R, typename F>
  static __device__ __forceinline__ void pv_apart(const Buf& b, int, const Prob (&p)[R], f32x4 (&acc)[R][VL], const F& in) {
#pragma unroll 1
    for (int key = 0; key < 32; ++key) {
      uint32_t mask[8];
      row_masks(key, mask);
#pragma unroll
      for (int e = 0; e < VL; ++e) {
        const w4 f = pick(b.v, e, mask);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          f32x4 s = {0.f, 0.f, 0.f, 0.f};
          s = Mma16<T>::run(f, only(p[r][0], mask), s);
          add_if(in(r, key), s, acc[r][e]);
        }
      }
    }
  }
  static __device__ __forceinline__ bool wild(const Buf& b, int) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    u16x2 top = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int w = 0; w < VL / 2; ++w) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, b.v[i][w] & 0x7fff7fffu));
    constexpr unsigned short kInf = __is_same(T, bf16) ? 0x7f80 : 0x7c00;
    return top.x >= kInf || top.y >= kInf;
  }
};

// Rows of fp32 values on the fp32 products (16x16x4): the four floats a lane loads
// of a K row are its operands in four of them, and a V element is one as it is.
template <int DL_> struct Rows32 {
  typedef float T;
  static constexpr int DL = DL_, VL = DL / 16, SUB = 1, QN = DL / 16;
  struct Buf {
    f32x4 k[2][QN];
    f32x4 v[8][VL / 4];
  };
  typedef f32x4 Query[QN];
  struct Prob {
    float p[8];
  };
  static constexpr bool kMx = false, kTerms = false;
  const char *kb, *vb;
  int koff[QN], voff[4][VL / 4];

  __device__ __forceinline__ void init(const Args& a, int h) {
    const int lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
    kb = static_cast<const char*>(a.k) + h * a.head;
    vb = static_cast<const char*>(a.v) + h * a.head;
#pragma unroll
    for (int j = 0; j < QN; ++j) koff[j] = 16 * j + 4 * g < a.d ? n * a.token + (16 * j + 4 * g) * 4 : kPad;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int h = 0; h < VL / 4; ++h) voff[i][h] = VL * n + 4 * h < a.d ? (4 * g + i) * a.token + (VL * n + 4 * h) * 4 : kPad;
  }
  static __device__ __forceinline__ void query(const Args& a, const T* row, bool live, Query& q) {
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int j = 0; j < QN; ++j) {
      q[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (live && 16 * j + 4 * g < a.d) q[j] = *reinterpret_cast<const f32x4*>(row + 16 * j + 4 * g);
      if (a.flip) q[j] = -q[j];
    }
  }
  __device__ __forceinline__ void load_k(const Look& l, int at, Buf& b) const {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const auto kr = tile_rsrc(kb, l.at, l.bytes, at + u);
#pragma unroll
      for (int j = 0; j < QN; ++j)
        b.k[u][j] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(kr, koff[j], 0, 0));
    }
  }
  __device__ __forceinline__ void load_v(const Look& l, int at, Buf& b) const {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const auto vr = tile_rsrc(vb, l.at, l.bytes, at + u);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int hh = 0; hh < VL / 4; ++hh)
          b.v[4 * u + i][hh] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(vr, voff[i][hh], 0, 0));
    }
  }
  static __device__ __forceinline__ void trim(Buf&, int) {}
  static __device__ __forceinline__ f32x4 score(const Buf& b, int t, const Query& q) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < QN; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_16x16x4f32(b.k[t][j][e], q[j][e], s, 0, 0, 0);
    return s;
  }
  static __device__ __forceinline__ void prob(const f32x4& lo, const f32x4& hi, Prob& p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p.p[i] = lo[i], p.p[4 + i] = hi[i];
  }
  template <int R>
  static __device__ __forceinline__ void pv(const Buf& b, int, const Prob (&p)[R], f32x4 (&acc)[R][VL]) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < VL; ++e)
#pragma unroll
        for (int r = 0; r < R; ++r)
          acc[r][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(b.v[i][e / 4][e % 4], p[r].p[i], acc[r][e], 0, 0, 0);
  }
  template <int R, typename F>
  static __device__ __forceinline__ void pv_apart(const Buf& b, int, const Prob (&p)[R], f32x4 (&acc)[R][VL], const F& in) {
#pragma unroll 1
    for (int key = 0; key < 32; ++key) {
      const bool mine = (int)((threadIdx.x & 63) >> 4) == (key & 15) >> 2;
      const int slot = 4 * (key >> 4) + (key & 3);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float pk = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) pk = mine && i == slot ? p[r].p[i] : pk;
#pragma unroll
        for (int e = 0; e < VL; ++e) {
          float v = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) v = mine && i == slot ? b.v[i][e / 4][e % 4] : v;
          add_if(in(r, key), __builtin_amdgcn_mfma_f32_16x16x4f32(v, pk, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0), acc[r][e]);
        }
      }
    }
  }
  static __device__ __forceinline__ bool wild(const Buf& b, int) {
    bool w = false;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < VL; ++e) w = w || !(fabsf(b.v[i][e / 4][e % 4]) < INFINITY);
    return w;
  }
};

// Rows of MXFP4 codes, 64 or 128 keys a step. A lane's K piece is DL / 4 consecutive
// channels (16 bytes are one block of 32), a V piece VL, inside one block. They become
// bf16, exactly, in registers; q and P are as many bf16 terms as their type has bits
// for (bf16 one, fp16 two, fp32 three), and P of bf16 two as well, so nothing is rounded on the way.
template <typename T_, int DL_> struct RowsMx {
  typedef T_ T;
  static constexpr int TERMS = sizeof(T) == 4 ? 3 : (__is_same(T, bf16) ? 1 : 2), PTERMS = sizeof(T) == 4 ? 3 : 2;
  static constexpr int DL = DL_, VL = DL / 16, QN = DL / 32;
  static constexpr int SUB = DL <= 128 && TERMS == 1 ? 4 : 2, NT = 2 * SUB;
  static constexpr bool kMx = true, kTerms = false;
  static constexpr int KW = DL >= 128 ? 4 : 2;     // words of codes in a K piece
  static constexpr int KP = DL >= 128 ? DL / 128 : 1;  // K pieces of a row in a lane
  static constexpr int VW = VL >= 8 ? VL / 8 : 1;  // words of codes of a V row in a lane (half a word at DL 64)
  struct Buf {
    uint32_t k[NT][KP][KW];
    uint32_t ke[NT][KP];  // scale bytes
    uint32_t v[4 * NT][VW];
    uint32_t ve[NT];  // scale bytes of the lane's four keys of each tile
  };
  typedef w4 Query[QN][TERMS];
  typedef w4 Prob[PTERMS];
  const char *kb, *vb, *kse_b, *vse_b;
  int scale_bytes;  // from a tile's first scale to behind its last
  int koff[KP], kse[KP], voff[4], vse;

  // channel of K piece word: product j takes these eight channels of a row from lane group g
  static __device__ __forceinline__ int channel(int j, int g) {
    return DL >= 128 ? 128 * (j / 4) + 32 * g + 8 * (j % 4) : 16 * g + 8 * j;
  }
  __device__ __forceinline__ void init(const Args& a, int h) {
    const int lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
    kb = static_cast<const char*>(a.k) + h * a.head;
    vb = static_cast<const char*>(a.v) + h * a.head;
    kse_b = reinterpret_cast<const char*>(a.ks) + h * a.shead;
    vse_b = reinterpret_cast<const char*>(a.vs) + h * a.shead;
    scale_bytes = (a.d / 32 - 1) * a.sblock + 16;
#pragma unroll
    for (int p = 0; p < KP; ++p) {
      const int c = channel(4 * p, g);
      koff[p] = c < a.d ? n * a.token + c / 2 : kPad;
      kse[p] = c < a.d ? (c / 32) * a.sblock + n : kPad;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) voff[i] = VL * n < a.d ? (4 * g + i) * a.token + VL * n / 2 : kPad;
    vse = VL * n < a.d ? (VL * n / 32) * a.sblock + 4 * g : kPad;
  }
  static __device__ __forceinline__ void query(const Args& a, const T* row, bool live, Query& q) {
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int j = 0; j < QN; ++j) {
      const int c = channel(j, g);
      Lane<T, 8> raw;
#pragma unroll
      for (int i = 0; i < Lane<T, 8>::kVectors; ++i) reinterpret_cast<w4*>(raw.v)[i] = w4{0, 0, 0, 0};
      if (live && c < a.d) raw = ld_lane<T, 8>(row + c);
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = a.flip ? -to_f32(raw.v[i]) : to_f32(raw.v[i]);
      terms_of<bf16, TERMS>(x, q[j]);
    }
  }
  __device__ __forceinline__ void load_k(const Look& l, int at, Buf& b) const {
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const auto kr = paged::tile_rsrc(kb, l.at, l.bytes, at + u);
      const auto sr = rsrc_of(kse_b + lane64(l.scales, at + u), (l.there >> (at + u)) & 1 ? scale_bytes : 0);
#pragma unroll
      for (int p = 0; p < KP; ++p) {
        if constexpr (KW == 4) {
          const w4 x = __builtin_amdgcn_raw_buffer_load_b128(kr, koff[p], 0, 0);
#pragma unroll
          for (int w = 0; w < 4; ++w) b.k[u][p][w] = x[w];
        } else {
          const w2 x = __builtin_amdgcn_raw_buffer_load_b64(kr, koff[p], 0, 0);
          b.k[u][p][0] = x.x, b.k[u][p][1] = x.y;
        }
        b.ke[u][p] = __builtin_amdgcn_raw_buffer_load_b8(sr, kse[p], 0, 0);
      }
    }
  }
  __device__ __forceinline__ void load_v(const Look& l, int at, Buf& b) const {
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const auto vr = paged::tile_rsrc(vb, l.at, l.bytes, at + u);
      const auto sr = rsrc_of(vse_b + lane64(l.scales, at + u), (l.there >> (at + u)) & 1 ? scale_bytes : 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t(&to)[VW] = b.v[4 * u + i];
        if constexpr (VL == 4) {
          to[0] = __builtin_amdgcn_raw_buffer_load_b16(vr, voff[i], 0, 0);
        } else if constexpr (VL == 8) {
          to[0] = __builtin_amdgcn_raw_buffer_load_b32(vr, voff[i], 0, 0);
        } else {
          const w2 x = __builtin_amdgcn_raw_buffer_load_b64(vr, voff[i], 0, 0);
          to[0] = x.x, to[1] = x.y;
        }
      }
      b.ve[u] = __builtin_amdgcn_raw_buffer_load_b32(sr, vse, 0, 0);
    }
  }
  // The scales of keys behind the last one, whatever they are, as if their rows were
  // zeros; `rows`: visible keys from the step's first on.
  static __device__ __forceinline__ void trim(Buf& b, int rows) {
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const int n = min(max(rows - 16 * u - 4 * g, 0), 4);
      b.ve[u] &= n == 4 ? 0xffffffffu : (1u << (8 * n)) - 1u;
    }
  }
  static __device__ __forceinline__ f32x4 score(const Buf& b, int t, const Query& q) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < QN; ++j) {
      const int p = DL >= 128 ? j / 4 : 0, w = DL >= 128 ? j % 4 : j;
      const w4 f = __builtin_bit_cast(w4, mx::decode8_bf16(b.k[t][p][w], mx::scale_of(b.ke[t][p])));
#pragma unroll
      for (int m = 0; m < TERMS; ++m) s = Mma16<bf16>::run(f, q[j][m], s);
    }
    return s;
  }
  static __device__ __forceinline__ void prob(const f32x4& lo, const f32x4& hi, Prob& p) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = lo[i], x[4 + i] = hi[i];
    terms_of<bf16, PTERMS>(x, p);
  }
  // The values of tiles 2 u and 2 u + 1 as bf16, VL to a row
  static __device__ __forceinline__ void decode(const Buf& b, int u, uint32_t (&v)[8][VL / 2]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = 8 * u + i;
      const float s = mx::scale_of((b.ve[2 * u + i / 4] >> (8 * (i % 4))) & 255u);
      if constexpr (VL == 4) {
        const mx::bf16x2 x = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(b.v[at][0], s, 0);
        const mx::bf16x2 y = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(b.v[at][0], s, 1);
        v[i][0] = __builtin_bit_cast(uint32_t, x), v[i][1] = __builtin_bit_cast(uint32_t, y);
      } else {
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          const uint4 x = mx::decode8_bf16(b.v[at][w], s);
          v[i][4 * w] = x.x, v[i][4 * w + 1] = x.y, v[i][4 * w + 2] = x.z, v[i][4 * w + 3] = x.w;
        }
      }
    }
  }
  template <int R>
  static __device__ __forceinline__ void pv(const Buf& b, int u, const Prob (&p)[R], f32x4 (&acc)[R][VL]) {
    uint32_t v[8][VL / 2];
    decode(b, u, v);
#pragma unroll
    for (int e = 0; e < VL; ++e) {
      const w4 f = pick(v, e);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int m = 0; m < PTERMS; ++m) acc[r][e] = Mma16<bf16>::run(f, p[r][m], acc[r][e]);
    }
  }
  template <int R, typename F>
  static __device__ __forceinline__ void pv_apart(const Buf& b, int u, const Prob (&p)[R], f32x4 (&acc)[R][VL], const F& in) {
    uint32_t v[8][VL / 2];
    decode(b, u, v);
#pragma unroll 1
    for (int key = 0; key < 32; ++key) {
      uint32_t mask[8];
      row_masks(key, mask);
#pragma unroll
      for (int e = 0; e < VL; ++e) {
        const w4 f = pick(v, e, mask);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int m = 0; m < PTERMS; ++m) s = Mma16<bf16>::run(f, only(p[r][m], mask), s);
          add_if(in(r, key), s, acc[r][e]);
        }
      }
    }
  }
  static __device__ __forceinline__ bool wild(const Buf& b, int u) {  // a scale of 255
    bool w = false;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) w = w || ((b.ve[2 * u + t] >> (8 * i)) & 255u) == 255u;
    return w;
  }
};

// Four consecutive outputs, each rounded once
template <typename T> __device__ __forceinline__ void store4(T* to, const f32x4& v) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(to) = v;
  else *reinterpret_cast<w2*>(to) = w2{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
}

// Zeros for the tokens that no sequence holds.
template <typename T> __device__ __forceinline__ void zero_others(const Args& a) {
  if (!a.cu) return;
  const int first = min(max(a.cu[0], 0), a.total), last = min(max(a.cu[a.seqs], first), a.total);
  for (int64_t i = blockIdx.x; i < first + a.total - last; i += gridDim.x) {
    T* row = static_cast<T*>(a.o) + (i < first ? i : i - first + last) * (int64_t)a.heads * a.d;
    for (int j = threadIdx.x; j < a.heads * a.d; j += blockDim.x) row[j] = from_f32<T>(0.f);
  }
}

// What the joining kernel reads: the row tiles there are, and of a tile of more than one
// chunk its first block and its rows.
__device__ __forceinline__ void note(const Args& a, const Item& it, int x, int h, int row0, int rows) {
  if (!a.split || h != 0 || it.chunk != 0 || threadIdx.x != 0 || it.tiles_base + it.tile >= a.tiles) return;
  int* m = a.meta + 1 + 4 * (int64_t)(it.tiles_base + it.tile);
  m[0] = x;
  m[1] = it.splits;
  m[2] = it.s.start * a.group + row0;  // the tile's first row among all rows of a kv head
  m[3] = rows;
}

// ---------------------------------------------------------------- the kernel of few rows

// SPLIT: the block's waves hold the same 16 R rows and take the steps of the chunk in
// turn, their sums joined in LDS at the end. Otherwise each wave has 16 R rows of its
// own and walks the whole chunk.
template <class C, int R, bool SPLIT> struct Shape {
  static constexpr int kRows = 16 * R * (SPLIT ? 1 : kWaves);
};

// Waves a SIMD holds: what the registers of a step's rows allow.
template <class C, int R> constexpr int kWavesPerEu = C::DL > 128 || R * sizeof(typename C::Buf) > 512 ? 1 : 2;

template <class C, int R, bool SPLIT>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(kWavesPerEu<C, R>))) void
attn_paged_kernel(Args a) {
  typedef typename C::T T;
  constexpr int ROWS = Shape<C, R, SPLIT>::kRows, VL = C::VL, DL = C::DL;
  constexpr int TILES = 2 * C::SUB, KEYS = 16 * TILES;  // of a step
  constexpr int PER = 64 / TILES;  // steps whose pages are looked up at once
  constexpr int LROW = DL + 4;
  __shared__ __attribute__((aligned(16))) float lds_o[SPLIT ? kWaves * 16 * R * LROW : 4];
  __shared__ float lds_m[SPLIT ? kWaves * 16 * R : 1], lds_l[SPLIT ? kWaves * 16 * R : 1];
  const int h = (int)(blockIdx.x % (unsigned)a.kv_heads), x = (int)(blockIdx.x / (unsigned)a.kv_heads);
  const int lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  zero_others<T>(a);
  const Item it = find<ROWS>(a, x);
  if (a.split && blockIdx.x == 0 && threadIdx.x == 0) a.meta[0] = min(it.all_tiles, a.tiles);
  if (it.seq < 0) return;  // the whole block, before any barrier
  const int all_rows = it.s.n * a.group, row0 = it.tile * ROWS;
  const int rows = min(ROWS, all_rows - row0);
  const bool joined = it.splits > 1;
  note(a, it, x, h, row0, rows);

  // this wave's rows: limit[r], the keys row n of sub-tile r sees; rows past the end repeat the last
  const int w0 = row0 + (SPLIT ? 0 : wave * 16 * R);
  const int in_front = it.s.len - it.s.n;  // keys in front of the new tokens
  const auto limit_of = [&](int row) {
    return a.causal ? max(0, in_front + token_of(a, min(row, all_rows - 1)) + 1) : it.s.len;
  };
  C cache;
  cache.init(a, h);
  typename C::Query q[R];
  int limit[R];
  const int k0 = (int)min((int64_t)it.chunk * it.keys, (int64_t)it.s.len);
  const int chunk_end = (int)min((int64_t)k0 + it.keys, (int64_t)it.s.len);
  const int k1 = min(chunk_end, limit_of(w0 + 16 * R - 1));
  const int low = min(limit_of(w0), chunk_end);  // keys below are seen by every row
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = w0 + 16 * r + n;
    const bool live = row < all_rows;
    const int token = live ? token_of(a, row) : 0, head = h * a.group + (live ? row - token * a.group : 0);
    C::query(a, static_cast<const T*>(a.q) + (it.s.start + token) * a.qt + head * a.qh, live, q[r]);
    limit[r] = min(limit_of(row), k1);
  }

  f32x4 acc[R][VL];
  float m[R], l[R];
  bool seen[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
    seen[r] = false;
#pragma unroll
    for (int e = 0; e < VL; ++e) acc[r][e] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // steps wave, wave + kWaves, ... of the chunk, or all of them
  const int steps = k1 > k0 ? (k1 - k0 + KEYS - 1) / KEYS : 0;
  const int own = SPLIT ? (steps - wave + kWaves - 1) / kWaves : (w0 < all_rows ? steps : 0);
  const auto step_of = [&](int i) { return SPLIT ? wave + kWaves * i : i; };
  const auto look = [&](int first) {
    const int64_t key = (int64_t)k0 + (int64_t)step_of(first + lane / TILES) * KEYS + 16 * (lane % TILES);
    return look_up<C::kMx>(a, it.seq, key, k1);
  };

  // One set of registers for a step's keys and values: the next step's keys are asked for
  // once the scores are made of this one's, its values once the products are.
  typename C::Buf b;
  Look lk;
  if (own > 0) {
    lk = look(0);
    cache.load_k(lk, 0, b);
    cache.load_v(lk, 0, b);
  }
  constexpr uint64_t kAll = (1ull << TILES) - 1;
  bool left = false;
  for (int i = 0; i < own; ++i) {
    const int key0 = k0 + step_of(i) * KEYS;
    const unsigned there = (unsigned)((lk.there >> (i % PER * TILES)) & kAll);
    const bool whole = key0 + KEYS <= low && ((lk.whole >> (i % PER * TILES)) & kAll) == kAll;
    f32x4 s[R][TILES];
    float top[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int u = 0; u < TILES; ++u) s[r][u] = C::score(b, u, q[r]);
    const bool more = i + 1 < own;
    if (more) {
      if ((i + 1) % PER == 0) lk = look(i + 1);
      cache.load_k(lk, (i + 1) % PER * TILES, b);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (!whole) {
#pragma unroll
        for (int u = 0; u < TILES; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bool in = ((there >> u) & 1) != 0 && key0 + 16 * u + 4 * g + j < limit[r];
            s[r][u][j] = in ? s[r][u][j] : -INFINITY;
            seen[r] |= in;
          }
      } else {
        seen[r] = true;
      }
      top[r] = -INFINITY;
#pragma unroll
      for (int u = 0; u < TILES; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) top[r] = fmaxf(top[r], s[r][u][j]);
    }
    bool over = false;
#pragma unroll
    for (int r = 0; r < R; ++r) over = over || top[r] * a.c > m[r] + kLag;
    if (__any(over)) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float t1 = fmaxf(top[r], __shfl_xor(top[r], 16, 64));
        t1 = fmaxf(t1, __shfl_xor(t1, 32, 64));
        const float now = fmaxf(m[r], t1 * a.c);
        const float f = now == m[r] ? 1.f : __builtin_amdgcn_exp2f(m[r] - now);
        m[r] = now;
        l[r] *= f;
#pragma unroll
        for (int e = 0; e < VL; ++e) acc[r][e] *= f;
      }
    }
    if (!whole) C::trim(b, k1 - key0);
#pragma unroll
    for (int u = 0; u < C::SUB; ++u) {
      typename C::Prob p[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float base = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r][2 * u + v][j], a.c, -base));
            s[r][2 * u + v][j] = e;
            l[r] += e;
          }
        C::prob(s[r][2 * u], s[r][2 * u + 1], p[r]);
      }
      // Where some rows see a key that others do not, an Inf or a NaN among the values must
      // stay out of the others (0 times it is a NaN): such steps are left for the loop below.
      // So are they where P has two terms (kTerms) and a value may be an Inf.
      if ((C::kTerms || (!whole && key0 + KEYS > low)) && __any(C::wild(b, u))) left = true;
      else C::template pv<R>(b, u, p, acc);
    }
    if (more) cache.load_v(lk, (i + 1) % PER * TILES, b);
  }

  // The values left: one key at a time, added to the rows that see it. (Apart from the loop
  // above, whose registers this took when it was part of it.)
  if (left)
    for (int i = 0; i < own; ++i) {
      const int key0 = k0 + step_of(i) * KEYS;
      if (!C::kTerms && key0 + KEYS <= low) continue;
      lk = look(i);
      cache.load_k(lk, 0, b);
      cache.load_v(lk, 0, b);
      C::trim(b, k1 - key0);
#pragma unroll
      for (int u = 0; u < C::SUB; ++u) {
        if (!__any(C::wild(b, u))) continue;
        typename C::Prob p[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float base = m[r] == -INFINITY ? 0.f : m[r];
          f32x4 s[2];
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            s[v] = C::score(b, 2 * u + v, q[r]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const bool in = ((lk.there >> (2 * u + v)) & 1) && key0 + 32 * u + 16 * v + 4 * g + j < limit[r];
              s[v][j] = in ? __builtin_amdgcn_exp2f(__builtin_fmaf(s[v][j], a.c, -base)) : 0.f;
            }
          }
          C::prob(s[0], s[1], p[r]);
        }
        C::template pv_apart<R>(b, u, p, acc, [&](int r, int key) { return key0 + 32 * u + key < limit[r]; });
      }
    }

  // the rows' sums over the four lanes that share each
#pragma unroll
  for (int r = 0; r < R; ++r) {
    l[r] += __shfl_xor(l[r], 16, 64);
    l[r] += __shfl_xor(l[r], 32, 64);
    const uint64_t any = __ballot(seen[r]);
    const bool had = ((any >> n) | (any >> (n + 16)) | (any >> (n + 32)) | (any >> (n + 48))) & 1;
    // a row with no key at all is told from one whose scores are all -Inf (0 / 0) by its maximum
    m[r] = had ? fmaxf(m[r], -3.4028235e38f) : -INFINITY;
  }
  const int64_t place = ((int64_t)x * a.kv_heads + h) * a.rows;  // this block's partial rows
  if constexpr (SPLIT) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int at = wave * 16 * R + 16 * r + n;
      if (g == 0) {
        lds_m[at] = m[r];
        lds_l[at] = l[r];
      }
      if (16 * r + n < rows) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < VL; e += 4)
            *reinterpret_cast<f32x4*>(&lds_o[at * LROW + VL * (4 * g + c) + e]) =
                f32x4{acc[r][e][c], acc[r][e + 1][c], acc[r][e + 2][c], acc[r][e + 3][c]};
      }
    }
    __syncthreads();
    const int quads = a.d / 4;
    for (int i = threadIdx.x; i < rows * quads; i += kThreads) {
      const int row = i / quads, d = (i - row * quads) * 4;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) top = fmaxf(top, lds_m[w * 16 * R + row]);
      const float base = top == -INFINITY ? 0.f : top;
      f32x4 sum = {0.f, 0.f, 0.f, 0.f};
      float den = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const int at = w * 16 * R + row;
        const float f = __builtin_amdgcn_exp2f(lds_m[at] - base);
        sum += *reinterpret_cast<const f32x4*>(&lds_o[at * LROW + d]) * f;
        den += lds_l[at] * f;
      }
      if (joined) {
        *reinterpret_cast<f32x4*>(a.part + (place + row) * a.d + d) = sum;
        if (d == 0) {
          a.ml[(place + row) * 2] = top;
          a.ml[(place + row) * 2 + 1] = den;
        }
      } else {
        const int full = row0 + row;
        T* to = row_of<T>(a, it.s.start, h, full) + d;
        store4(to, sum * (top == -INFINITY ? 0.f : 1.f / den));
      }
    }
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = w0 + 16 * r + n - row0;  // in the block's tile
      if (row >= rows) continue;
      const int full = row0 + row;
      T* to = row_of<T>(a, it.s.start, h, full);
      const float inv = m[r] == -INFINITY ? 0.f : 1.f / l[r];
      if (joined && g == 0) {
        a.ml[(place + row) * 2] = m[r];
        a.ml[(place + row) * 2 + 1] = l[r];
      }
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int e = 0; e < VL; e += 4) {
          const int d = VL * (4 * g + c) + e;
          if (d >= a.d) continue;
          const f32x4 v = {acc[r][e][c], acc[r][e + 1][c], acc[r][e + 2][c], acc[r][e + 3][c]};
          if (joined) *reinterpret_cast<f32x4*>(a.part + (place + row) * a.d + d) = v;
          else store4(to + d, v * inv);
        }
    }
  }
}

// Joins the chunks of split row tiles: a block takes kJoinRows rows of a tile (one where a
// tile has at most 16), a thread four dims of every parts-th chunk of a row, where the
// rows leave threads for more than one part; parts are then added in their order.
constexpr int kJoinThreads = 256;
inline __host__ __device__ int join_rows(int rows) { return rows > 16 ? 8 : 1; }

template <typename T> __global__ __launch_bounds__(kJoinThreads) void attn_paged_join(Args a) {
  __shared__ f32x4 sums[kJoinThreads];
  __shared__ float dens[kJoinThreads];
  const int each = join_rows(a.rows), groups = (a.rows + each - 1) / each;
  const int from = (int)(blockIdx.x % (unsigned)groups) * each;
  const int h = (int)(blockIdx.x / (unsigned)groups % (unsigned)a.kv_heads);
  const int tile = (int)(blockIdx.x / (unsigned)groups / (unsigned)a.kv_heads);
  if (tile >= a.meta[0]) return;
  const int* m = a.meta + 1 + 4 * (int64_t)tile;
  const int first = m[0], splits = m[1], row0 = m[2], rows = m[3];
  if (splits <= 1 || from >= rows) return;  // the whole block, before any barrier
  if (first < 0 || splits > a.items - first || row0 < 0 || row0 > a.total * a.group - rows || rows > a.rows) return;
  const int quads = a.d / 4, slots = kJoinThreads / quads;
  int parts = 1;
  while (2 * parts * each <= slots && 2 * parts <= splits) parts *= 2;
  const int q = threadIdx.x % quads, slot = threadIdx.x / quads, part = slot % parts;
  const int at_once = slots / parts, end = min(from + each, rows);
  for (int base_row = from; base_row < end; base_row += at_once) {
    const int row = base_row + slot / parts;
    const bool mine = slot < at_once * parts && row < end;
    float top = -INFINITY;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    float den = 0.f;
    if (mine) {
      const int64_t step = (int64_t)a.kv_heads * a.rows, at = ((int64_t)first * a.kv_heads + h) * a.rows + row;
      const float* ml = a.ml + 2 * at;
      const float* part_sum = a.part + at * a.d + 4 * q;
#pragma unroll 8
      for (int s = 0; s < splits; ++s) top = fmaxf(top, ml[2 * s * step]);
      const float base = top == -INFINITY ? 0.f : top;
#pragma unroll 4
      for (int s = part; s < splits; s += parts) {
        const float f = __builtin_amdgcn_exp2f(ml[2 * s * step] - base);
        sum += *reinterpret_cast<const f32x4*>(part_sum + s * step * a.d) * f;
        den += ml[2 * s * step + 1] * f;
      }
    }
    sums[threadIdx.x] = sum;
    dens[threadIdx.x] = den;
    __syncthreads();
    if (mine && part == 0) {
      for (int i = 1; i < parts; ++i) {
        sum += sums[threadIdx.x + i * quads];
        den += dens[threadIdx.x + i * quads];
      }
      store4(row_of<T>(a, 0, h, row0 + row) + 4 * q, sum * (top == -INFINITY ? 0.f : 1.f / den));
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- host side

// Rows of a block's tile: 16 that the waves split the keys of, or 128 that they share out,
// where a sequence has more than 32 rows on average and the work is enough for the fewer
// blocks: row tiles of 16 times keys (as many as the table holds) past 768 a block that
// runs at once over 16-bit rows, 2048 over 4 bits and in fp32. One sequence of 128 rows a
// kv head, 8 of them, 128 dims, bf16: 9 us at 16 rows, 16 at 128 over 256 keys, 16 and 26
// over 1024, 34 and 30 over 8192; eight of 1024 rows over 8192: 1173 and 333; into 4 bits
// with fp16 q 27 and 40, and 695 and 496. Over 270 such calls the choice costs 1 to 4 % of
// the better side, always 128 rows 21 to 91 %. fp32 q over MXFP4 has three terms of q and P,
// which leave a wave no second one beside it: 16 rows are as fast or faster (eight of 1024
// rows over 8192 keys, 128 dims: 800 us against 959; 256 dims, 3 x 300 tokens over 12000
// keys, 16/4 heads: 802, 903) but for 129 to 192 dims, for which that kernel has only rows
// of 256 (192 dims: 815, 616).
struct Plan {
  bool wide;
  int rows;           // of a tile
  int64_t tiles;      // row tiles at most
  int64_t items;      // blocks a kv head at most
  bool split;
  int min_chunk, target, at_once;
  int part_rows;
  int64_t part_bytes, ml_bytes, meta_bytes;
};

inline Plan plan_of(int64_t seqs, int64_t total, bool packed, int64_t kv_heads, int64_t group, int64_t head_dim,
                    int64_t capacity, bool f32, bool mxfp4) {
  Plan p{};
  const int64_t rows = total * group;
  p.at_once = 2 * cu_count();  // eight waves a CU, what their registers allow
  p.wide = packed && rows > 32 * seqs && (double)(rows * kv_heads / 16) * capacity > p.at_once * (f32 || mxfp4 ? 2048. : 768.) &&
           !(f32 && mxfp4 && (head_dim <= 128 || head_dim > 192));
  p.rows = p.wide ? (f32 && !mxfp4 && head_dim > 128 ? 64 : 128) : 16;
  p.tiles = packed ? rows / p.rows + seqs : seqs * ((group + p.rows - 1) / p.rows);
  if (p.tiles < 1) p.tiles = 1;
  p.min_chunk = 512;
  p.target = (int)((p.at_once + kv_heads - 1) / kv_heads);
  p.split = capacity > p.min_chunk && (!p.wide || p.tiles * kv_heads < p.at_once);
  p.items = p.tiles;
  if (p.split) {  // a chunk is at least a kParts-th of an even share, and min_chunk keys
    const int64_t most = p.tiles * ((capacity + p.min_chunk - 1) / p.min_chunk);
    p.items = most < p.tiles + kParts * p.target ? most : p.tiles + kParts * p.target;
  }
  p.part_rows = packed ? p.rows : (int)(group < p.rows ? group : p.rows);
  if (p.split) {
    p.part_bytes = (p.items * kv_heads * p.part_rows * head_dim * 4 + 255) / 256 * 256;
    p.ml_bytes = (p.items * kv_heads * p.part_rows * 8 + 255) / 256 * 256;
    p.meta_bytes = ((1 + 4 * p.tiles) * 4 + 255) / 256 * 256;
  }
  return p;
}

inline int log2_of(int64_t n) {  // -1: not a power of two
  for (int i = 0; i < 31; ++i)
    if (n == (int64_t)1 << i) return i;
  return -1;
}

inline int check_plan(const char* who, const Plan& p, int64_t kv_heads) {
  if (p.items * kv_heads > INT32_MAX || (p.split && p.tiles * kv_heads * p.part_rows > INT32_MAX))
    return fail(PK_ERR_UNSUPPORTED, "%s: grid too large", who);
  return PK_OK;
}

inline void set_plan(Args& a, const Plan& p) {
  a.rows = p.part_rows;
  a.items = (int)p.items;
  a.tiles = (int)p.tiles;
  a.split = p.split;
  a.min_chunk = p.min_chunk;
  a.target = (float)p.target;
  a.at_once = (float)p.at_once;
}

template <typename T> void launch_join(const Args& a, const Plan& p, hipStream_t s) {
  if (p.split)
    hipLaunchKernelGGL(attn_paged_join<T>,
                       dim3((unsigned)(p.tiles * a.kv_heads * ((a.rows + join_rows(a.rows) - 1) / join_rows(a.rows)))),
                       dim3(kJoinThreads), 0, s, a);
}

template <class C, int R, bool SPLIT> int launch(Args a, const Plan& p, hipStream_t s, const char* who) {
  set_plan(a, p);
  hipLaunchKernelGGL((attn_paged_kernel<C, R, SPLIT>), dim3((unsigned)(p.items * a.kv_heads)),
                     dim3(kThreads), 0, s, a);
  launch_join<typename C::T>(a, p, s);
  return launched(who);
}

// Checks and fields that both entry points share. strides: q (token, head), then the
// cache's k and v (page, head, token), in elements of `bytes` each; PK_OK with *empty:
// nothing to do.
inline int paged_args(const char* who, Args& a, const int64_t* strides, int64_t seqs, int64_t total, int64_t q_heads,
                      int64_t kv_heads, int64_t head_dim, int64_t num_pages, int64_t page_size, int64_t table_width,
                      int64_t table_stride, float softmax_scale, int causal, int dtype, bool mxfp4, void* workspace,
                      int64_t workspace_bytes, Plan& p, bool* empty) {
  *empty = false;
  if (seqs < 0 || total < 0 || q_heads < 0 || kv_heads < 0 || num_pages < 0 || table_width < 0)
    return fail(PK_ERR_INVALID, "%s: negative size", who);
  if (!known_dtype(dtype)) return fail(PK_ERR_UNSUPPORTED, "%s: dtype code %d (bf16/fp16/fp32 only)", who, dtype);
  const int unit = mxfp4 ? 32 : 8;
  if (head_dim <= 0 || head_dim > 256 || head_dim % unit != 0)
    return fail(PK_ERR_UNSUPPORTED, "%s: head_dim=%lld (a multiple of %d up to 256)", who, (long long)head_dim, unit);
  if (page_size < 16 || page_size % 16 != 0 || page_size > (1 << 20))
    return fail(PK_ERR_UNSUPPORTED, "%s: page_size=%lld is not a multiple of 16 up to 2^20", who, (long long)page_size);
  if (!isfinite(softmax_scale)) return fail(PK_ERR_INVALID, "%s: softmax_scale is not finite", who);
  if (total == 0 || q_heads == 0) {
    *empty = true;
    return PK_OK;
  }
  if (kv_heads == 0 || q_heads % kv_heads != 0)
    return fail(PK_ERR_INVALID, "%s: q_heads=%lld is not a multiple of kv_heads=%lld", who, (long long)q_heads,
                (long long)kv_heads);
  if (seqs > (1 << 24) || total * q_heads > INT32_MAX || num_pages > INT32_MAX || table_width * page_size > (1 << 30))
    return fail(PK_ERR_UNSUPPORTED, "%s: shape too large", who);
  if (!a.cu && seqs != total) return fail(PK_ERR_INVALID, "%s: one token a sequence, but %lld tokens and %lld sequences", who,
                                          (long long)total, (long long)seqs);
  const bool cached = num_pages > 0 && table_width > 0 && seqs > 0;
  if (!a.q || !a.o || !strides || (seqs > 0 && (!a.lens || (table_width > 0 && !a.table))) ||
      (cached && (!a.k || !a.v)) ||
      (cached && mxfp4 && (!a.ks || !a.vs)))
    return fail(PK_ERR_INVALID, "%s: null pointer", who);
  if (!aligned16(a.q) || !aligned16(a.o) || !aligned16(a.k) || !aligned16(a.v))
    return fail(PK_ERR_INVALID, "%s: q, o and the cache must be 16-byte aligned", who);
  const int e = elem_size(dtype), held = mxfp4 ? 1 : e;
  // how many of each dimension there are: the stride of a lone one is not looked at
  const int64_t counts[8] = {total, q_heads, num_pages, kv_heads, page_size, num_pages, kv_heads, page_size};
  for (int i = 0; i < 8; ++i)
    if (counts[i] > 1 && (strides[i] < 0 || strides[i] * (i < 2 ? e : held) % 16 != 0))
      return fail(PK_ERR_INVALID, "%s: stride %d = %lld is not a non-negative multiple of 16 bytes", who, i,
                  (long long)strides[i]);
  const int64_t row = mxfp4 ? head_dim / 2 : head_dim * e;
  if (strides[4] * held * 16 + row > INT32_MAX)
    return fail(PK_ERR_UNSUPPORTED, "%s: 16 rows of a page span more than 2 GiB", who);
  for (int i = 2; i < 5; ++i)
    if (counts[i] > 1 && strides[i] != strides[i + 3])
      return fail(PK_ERR_UNSUPPORTED, "%s: the key and the value cache have different strides", who);
  a.qt = strides[0], a.qh = strides[1];
  a.page = strides[2] * held, a.head = strides[3] * held, a.token = (int)(strides[4] * held);
  a.elem = e;
  a.tpp_shift = log2_of(page_size / 16);
  a.group_shift = log2_of(q_heads / kv_heads);
  a.table_stride = table_stride;
  a.width = (int)table_width;
  a.pages = (int)num_pages;
  a.tiles_per_page = (int)(page_size / 16);
  a.seqs = (int)seqs;
  a.total = (int)total;
  a.heads = (int)q_heads;
  a.kv_heads = (int)kv_heads;
  a.group = (int)(q_heads / kv_heads);
  a.d = (int)head_dim;
  a.causal = causal;
  a.c = fmaxf(fabsf(softmax_scale) * 1.4426950408889634f, 1e-30f);
  a.flip = softmax_scale < 0.f ? 0x80008000u : 0u;
  p = plan_of(seqs, total, a.cu != nullptr, kv_heads, a.group, head_dim, table_width * page_size,
              dtype == PK_F32, mxfp4);
  const int status = check_plan(who, p, kv_heads);
  if (status != PK_OK) return status;
  const int64_t need = p.part_bytes + p.ml_bytes + p.meta_bytes;
  if (need > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < need))
    return fail(PK_ERR_INVALID, "%s: workspace of %lld bytes, %lld (16-byte aligned) needed", who,
                (long long)workspace_bytes, (long long)need);
  char* w = static_cast<char*>(workspace);
  a.part = reinterpret_cast<float*>(w);
  a.ml = reinterpret_cast<float*>(w + p.part_bytes);
  a.meta = reinterpret_cast<int*>(w + p.part_bytes + p.ml_bytes);
  return PK_OK;
}

}  // namespace paged
}  // namespace pk
