// Attention over a paged cache for many rows (prompts, chunks of them): attn_paged.h's
// work items at 128 rows, four waves of 32, over key tiles of 32 that the block shares
// in LDS. 16-bit products of 32 x 32 x 16, on transposes as in attn_fwd.hip:
//   S^T (32 keys x 32 rows) = K . Q^T,  O^T (dims x 32 rows) += V^T . P^T
// with lane l holding row l % 32 and, of each tile's scores, keys 8 (r / 4) + 4 (l / 32) + r % 4.
//
// What bounds it are the products and the vector work beside them. A few rows read each
// K and V piece into registers straight from the cache; here four waves need the same
// tile, so it goes through LDS once a block: rows of 16-bit values by loads that write
// LDS directly, MXFP4 codes through registers, where they become bf16 (exactly) once a
// block and not once a wave. Each tile is two halves of 16 keys, which lie in one page
// each. LDS rows are unpadded, chunk c of row r at slot c ^ swz(r): a K fragment read
// takes the same chunk of 16 consecutive rows, which the swizzle spreads over the 16
// slots of a 256-byte bank window; V is read by transposing reads (attn_fwd.hip). Rows are
// laid out for 64, 96, 128, 192 or 256 dims: rows of 96 and 192 already start at four and
// two different places of the window, and swizzles of two and three bits do the rest.
//
// Step t turns S(t) into P(t), then runs O += V(t)^T P(t)^T and S(t + 1) = K(t + 1) Q^T as
// one sequence of products whose LDS fragments are read kRing products ahead; K(t + 2) and
// V(t + 1) are asked for at its start and there at its end, at one barrier a step.
//
// q and P enter as TERMS values of E (attn_paged.h): one where E is q's own type, as in the
// forward of whole sequences. P is then rounded once, by half a step of E at most, which
// many rows can bear beside the output's own rounding (bf16: 0.0023 of the values' size
// against 0.0017 from the output alone); a second term would be half as many products again.
//
// 4 x 8192 tokens of 32/8 heads of 128, causal, bf16: 2227 us, 988 TFLOP/s. Chunks of 2048
// tokens over 4096 to 8192 keys, four of them: 412 us, 821 TFLOP/s, the rest being the last
// of 880 blocks. 300 fp16 tokens over 20011 keys in MXFP4, 28/4 heads of 96: 226 us
// (20 more in rows of 128).
#pragma once

#include "attn_paged.h"

namespace pk {
namespace paged {

using attn::f32x16;
using attn::s16x4;

constexpr int kTile = 32;

template <int DL> __device__ __forceinline__ int k_swz(int r) {
  return DL == 96 ? (r >> 2) & 3 : (DL % 128 == 64 ? (r >> 1) & 7 : r & 15);
}
template <int DL> __device__ __forceinline__ int v_swz(int r) {
  return DL == 96 ? 0 : (DL % 128 == 64 ? 4 * ((r >> 1) & 1) : 4 * (r & 3));
}
// Element of a row that lies `dims` (a multiple of 16) behind the one at `at`: the bits that
// a swizzle reaches, below the lowest one set in DL, are flipped, and the others added.
template <int DL> __device__ __forceinline__ int behind(int at, int dims) {
  constexpr int LOW = (DL & -DL) - 1;
  return (at ^ (dims & LOW)) + (dims & ~LOW);
}

// Tiles of E in LDS, two of each (the step's and the next one's), and zeros in the place
// of values that a step leaves out
template <typename E, int DL> struct Shared {
  E k[2][kTile * DL];
  E v[3][kTile * DL];
};

// Staging of 16-bit rows: whole 16-byte slots, written by the load itself.
template <typename E, int DL> struct StageRows {
  static constexpr bool kMx = false;
  static constexpr int CH = DL / 8, NI = 16 * CH / 64;  // chunks of a row; wave instructions of a half tile
  static constexpr int OWN = (2 * NI + kWaves - 1) / kWaves;             // of both halves, a wave's
  static constexpr int PARTS = NI % kWaves == 0 ? NI / kWaves : OWN;  // different places in a half among them
  const char *kb, *vb;
  int wave, koff[PARTS], voff[PARTS];

  __device__ __forceinline__ void init(const Args& a, int h, int wave_) {
    wave = wave_;
    kb = static_cast<const char*>(a.k) + h * a.head;
    vb = static_cast<const char*>(a.v) + h * a.head;
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      const int s = ((wave + kWaves * p) % NI) * 64 + (threadIdx.x & 63), row = s / CH, pos = s % CH;
      const int kc = (pos ^ k_swz<DL>(row)) * 8, vc = (pos ^ v_swz<DL>(row)) * 8;
      koff[p] = kc < a.d ? row * a.token + kc * 2 : kPad;
      voff[p] = vc < a.d ? row * a.token + vc * 2 : kPad;
    }
  }
  __device__ __forceinline__ void fetch(const char* base, const int (&offs)[PARTS], const Look& l, int at, E* to) const {
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      const int id = wave + kWaves * i, half = id / NI, part = id % NI;  // half is the wave's own
      if (2 * NI % kWaves != 0 && id >= 2 * NI) break;
      const auto r = attn::make_rsrc_words(base + lane64(l.at, at + half), __builtin_amdgcn_readlane(l.bytes, at + half));
      attn::ld_lds16_asm(r, to + (half * 16 * CH + part * 64) * 8, offs[i % PARTS], 0);
    }
  }
  // The tile whose halves are lanes at and at + 1 of l, into LDS, asynchronously.
  __device__ __forceinline__ void fetch_k(const Look& l, int at, E* k) const { fetch(kb, koff, l, at, k); }
  __device__ __forceinline__ void fetch_v(const Look& l, int at, E* v) const { fetch(vb, voff, l, at, v); }
  // after the step: what was fetched lies in LDS
  __device__ __forceinline__ void store_k(int, E*) const { attn::lds_loads_landed(); }
  __device__ __forceinline__ void store_v(int, E*) const {}
};

// Staging of MXFP4 rows: a thread takes eight codes and their scale into registers, and
// makes 16 bytes of LDS of them after the step.
template <int DL> struct StageMx {
  typedef bf16 E;
  static constexpr bool kMx = true;
  static constexpr int CH = DL / 8, ALL = kTile * CH, OWN = (ALL + kThreads - 1) / kThreads;
  const char *kb, *vb, *ksb, *vsb;
  int scale_bytes;
  int off[OWN], soff[OWN];
  uint32_t kc[OWN], ke[OWN], vc[OWN], ve[OWN];

  static __device__ __forceinline__ int row(int i) { return (i * kThreads + (int)threadIdx.x) / CH; }
  static __device__ __forceinline__ int chunk(int i) { return (i * kThreads + (int)threadIdx.x) % CH; }
  // whether this wave has chunks i at all
  static __device__ __forceinline__ bool has(int i) {
    return ALL % kThreads == 0 || i * kThreads + (int)__builtin_amdgcn_readfirstlane(threadIdx.x) < ALL;
  }
  __device__ __forceinline__ void init(const Args& a, int h, int) {
    kb = static_cast<const char*>(a.k) + h * a.head;
    vb = static_cast<const char*>(a.v) + h * a.head;
    ksb = reinterpret_cast<const char*>(a.ks) + h * a.shead;
    vsb = reinterpret_cast<const char*>(a.vs) + h * a.shead;
    scale_bytes = (a.d / 32 - 1) * a.sblock + 16;
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      const int r = row(i) % 16, c = chunk(i);
      off[i] = 8 * c < a.d ? r * a.token + 4 * c : kPad;
      soff[i] = 8 * c < a.d ? (c / 4) * a.sblock + r : kPad;
    }
  }
  __device__ __forceinline__ void fetch(const char* rows, const char* scales, const Look& l, int at, uint32_t (&c)[OWN],
                                        uint32_t (&e)[OWN]) const {
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      if (!has(i)) break;
      const int half = __builtin_amdgcn_readfirstlane(row(i) / 16);  // 64 consecutive chunks lie in one half
      const int bytes = __builtin_amdgcn_readlane(l.bytes, at + half);
      c[i] = __builtin_amdgcn_raw_buffer_load_b32(rsrc_of(rows + lane64(l.at, at + half), bytes), off[i], 0, 0);
      e[i] = __builtin_amdgcn_raw_buffer_load_b8(rsrc_of(scales + lane64(l.scales, at + half), bytes > 0 ? scale_bytes : 0),
                                                 soff[i], 0, 0);
    }
  }
  __device__ __forceinline__ void fetch_k(const Look& l, int at, E*) { fetch(kb, ksb, l, at, kc, ke); }
  __device__ __forceinline__ void fetch_v(const Look& l, int at, E*) { fetch(vb, vsb, l, at, vc, ve); }
  // rows: visible keys of the tile; the scales behind them may be anything
  template <typename S>
  __device__ __forceinline__ void store(int rows, E* to, const uint32_t (&codes)[OWN], const uint32_t (&e)[OWN], const S& swz) const {
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      if (!has(i)) break;
      const int r = row(i);
      *reinterpret_cast<uint4*>(to + (r * CH + (chunk(i) ^ swz(r))) * 8) =
          mx::decode8_bf16(codes[i], mx::scale_of(r < rows ? e[i] : 0u));
    }
  }
  __device__ __forceinline__ void store_k(int rows, E* k) const {
    store(rows, k, kc, ke, [](int r) { return k_swz<DL>(r); });
  }
  __device__ __forceinline__ void store_v(int rows, E* v) const {
    store(rows, v, vc, ve, [](int r) { return v_swz<DL>(r); });
  }
};

// LDS fragments in flight ahead of the product that uses them
template <int DL> constexpr int kRing = DL > 128 ? 3 : 6;

// TERMS_Q, TERMS_P: values of E that q and P are the sums of.
template <typename T, typename E, int DL, int TERMS_Q, int TERMS_P, class Stage>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(DL > 128 || TERMS_Q > 2 ? 1 : 2))) void attn_paged_wide_kernel(
    Args a) {
  typedef typename attn::Mma<E>::frag Frag;
  constexpr int ROWS = 32 * kWaves, CH = DL / 8, KK = DL / 16, DT = DL / 32;
  constexpr int PER = 32;  // tiles whose pages are looked up at once: two halves each
  __shared__ __attribute__((aligned(16))) Shared<E, DL> lds;
  const int h = (int)(blockIdx.x % (unsigned)a.kv_heads), x = (int)(blockIdx.x / (unsigned)a.kv_heads);
  const int lane = threadIdx.x & 63, r32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  zero_others<T>(a);
  const Item it = find<ROWS>(a, x);
  if (a.split && blockIdx.x == 0 && threadIdx.x == 0) a.meta[0] = min(it.all_tiles, a.tiles);
  if (it.seq < 0) return;  // the whole block, before any barrier
  const int all_rows = it.s.n * a.group, row0 = it.tile * ROWS;
  const int rows = min(ROWS, all_rows - row0);
  const bool joined = it.splits > 1;
  note(a, it, x, h, row0, rows);

  const int in_front = it.s.len - it.s.n;
  const auto limit_of = [&](int row) {
    return a.causal ? max(0, in_front + token_of(a, min(row, all_rows - 1)) + 1) : it.s.len;
  };
  const int w0 = row0 + 32 * wave;
  const int k0 = (int)min((int64_t)it.chunk * it.keys, (int64_t)it.s.len);
  const int chunk_end = (int)min((int64_t)k0 + it.keys, (int64_t)it.s.len);
  const int k1 = min(chunk_end, limit_of(row0 + ROWS - 1));  // keys the block goes over
  const int low = min(limit_of(w0), chunk_end);              // keys every row of the wave sees
  const int limit = min(limit_of(w0 + r32), k1);

  Frag q[KK][TERMS_Q];
  {
    const int row = w0 + r32;
    const bool live = row < all_rows;
    const int token = live ? token_of(a, row) : 0, head = h * a.group + (live ? row - token * a.group : 0);
    const T* qr = static_cast<const T*>(a.q) + (it.s.start + token) * a.qt + head * a.qh;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const int c = 16 * kk + 8 * g;
      if constexpr (sizeof(T) == 2 && TERMS_Q == 1) {
        w4 raw = {0, 0, 0, 0};
        if (live && c < a.d) raw = *reinterpret_cast<const w4*>(qr + c);
        q[kk][0] = __builtin_bit_cast(Frag, raw ^ a.flip);
      } else {
        Lane<T, 8> raw;
#pragma unroll
        for (int i = 0; i < Lane<T, 8>::kVectors; ++i) reinterpret_cast<w4*>(raw.v)[i] = w4{0, 0, 0, 0};
        if (live && c < a.d) raw = ld_lane<T, 8>(qr + c);
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = a.flip ? -to_f32(raw.v[i]) : to_f32(raw.v[i]);
        w4 t[TERMS_Q];
        terms_of<E, TERMS_Q>(v, t);
#pragma unroll
        for (int m = 0; m < TERMS_Q; ++m) q[kk][m] = __builtin_bit_cast(Frag, t[m]);
      }
    }
  }
  f32x16 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[dt][r] = 0.f;
  float m = -INFINITY, l = 0.f;
  bool seen = false;

  Stage stage;
  stage.init(a, h, wave);
  // the compiler's own loads complete before the first load it does not see
  __builtin_amdgcn_s_waitcnt(0x0F70);
  const int steps = k1 > k0 ? (k1 - k0 + kTile - 1) / kTile : 0;
  const auto look = [&](int first) {
    return look_up<Stage::kMx>(a, it.seq, (int64_t)k0 + (int64_t)first * kTile + 16 * lane, k1);
  };
  // this lane's places in a tile: K fragment kk (keys r32, dims 16 kk + 8 g .. + 7) 16 kk
  // behind k_at, and V^T's transposing reads (key rows v_kr + 16 c + 8 h, dims 32 dt +
  // 16 ((lane >> 4) & 1) + 4 (lane & 3) .. + 3) 32 dt behind v_at
  const int k_at = (r32 * CH + (g ^ k_swz<DL>(r32))) * 8;
  const int v_kr = 4 * g + ((lane & 15) >> 2);
  const int v_at = v_kr * DL + (v_swz<DL>(v_kr) + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) * 8 + 4 * (lane & 1);
  // (from k_at and v_at in the step's buffers, which the compiler is kept from splitting into
  // an address for each kk and dt: registers that the loop does not have)
  const auto kfrag = [&](int k_now, int kk) -> Frag {
    return *reinterpret_cast<const Frag*>(&lds.k[0][0] + behind<DL>(k_now, 16 * kk));
  };
  const auto k_in = [&](int buf) {
    int k_now = k_at + buf * (kTile * DL);
    asm volatile("" : "+v"(k_now));
    return k_now;
  };
  const auto v_in = [&](int buf) {
    int v_now = v_at + buf * (kTile * DL);
    asm volatile("" : "+v"(v_now));
    return v_now;
  };
  const auto vfrag = [&](int v_now, int c, int dt) -> Frag {
    const E* at = &lds.v[0][0] + behind<DL>(v_now, 32 * dt);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((attn::lds_s4*)(at + 16 * c * DL));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((attn::lds_s4*)(at + (16 * c + 8) * DL));
    return __builtin_bit_cast(Frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  const auto scores = [&](int buf) {
    const int k_now = k_in(buf);
    f32x16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const Frag f = kfrag(k_now, kk);
#pragma unroll
      for (int n = 0; n < TERMS_Q; ++n) s = attn::Mma<E>::run(f, q[kk][n], s);
    }
    return s;
  };

  // Where some rows see a key that others do not, an Inf or a NaN among the values must
  // stay out of the others (0 times it is a NaN).
  const auto wild_tile = [&](const E* vb) {
    bool wild = false;
#pragma unroll 1
    for (int i = 0; i < DL / 16; ++i) {
      const w4 w = *reinterpret_cast<const w4*>(vb + (i * 64 + lane) * 8);
#pragma unroll
      for (int n = 0; n < 4; ++n) wild |= wild2<E>(w[n]);
    }
    return wild;
  };
  bool left = false;

  for (int i = threadIdx.x; i < kTile * DL / 8; i += kThreads) reinterpret_cast<w4*>(lds.v[2])[i] = w4{0, 0, 0, 0};
  Look lk;
  int first = 0;  // the tile of lane 0 of lk
  f32x16 s;
  if (steps > 0) {
    lk = look(0);
    __builtin_amdgcn_s_waitcnt(0x0F70);
    stage.fetch_k(lk, 0, lds.k[0]);
    stage.fetch_v(lk, 0, lds.v[0]);
    stage.store_k(k1 - k0, lds.k[0]);
    stage.store_v(k1 - k0, lds.v[0]);
    stage.fetch_k(lk, 2, lds.k[1]);
    stage.store_k(k1 - k0 - kTile, lds.k[1]);
    __syncthreads();
    s = scores(0);
    __syncthreads();  // K(0) is read; the first step overwrites it
  }
  for (int t = 0; t < steps; ++t) {
    const int key0 = k0 + t * kTile;
    if (t + 2 - first == PER) {
      lk = look(t);
      first = t;
      __builtin_amdgcn_s_waitcnt(0x0F70);
    }
    const int at = 2 * (t - first);
    // behind the last tile these read nothing
    stage.fetch_k(lk, at + 4, lds.k[t & 1]);
    stage.fetch_v(lk, at + 2, lds.v[(t + 1) & 1]);
    const bool whole = key0 + kTile <= low && ((lk.whole >> at) & 3u) == 3u;
    const E* vs = lds.v[t & 1];
    bool wild = false;
    if (!whole) {
      const unsigned there = (unsigned)(lk.there >> at) & 3u;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const bool in = (there & (1u << (r / 8))) && key0 + 8 * (r / 4) + 4 * g + r % 4 < limit;
        s[r] = in ? s[r] : -INFINITY;
        seen |= in;
      }
      if (key0 + kTile > low) wild = wild_tile(vs);
    } else {
      seen = true;
    }
    float top = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
    if (__any(top * a.c > m + kLag)) {
      const float now = fmaxf(m, fmaxf(top, __shfl_xor(top, 32, 64)) * a.c);
      const float f = now == m ? 1.f : __builtin_amdgcn_exp2f(m - now);
      m = now;
      l *= f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[dt] *= f;
    }
    const float base = m == -INFINITY ? 0.f : m;
    Frag p[2][TERMS_P];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        e[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * c + j], a.c, -base));
        l += e[j];
      }
      w4 w[TERMS_P];
      terms_of<E, TERMS_P>(e, w);
#pragma unroll
      for (int n = 0; n < TERMS_P; ++n) p[c][n] = __builtin_bit_cast(Frag, w[n]);
    }
    // the values of a wild tile are left for the loop below: zeros in their place (a branch
    // around the products cost the loop fourteen registers)
    const bool out = __any(wild);
    left |= out;
    constexpr int N = 2 * KK, RING = kRing<DL> < N ? kRing<DL> : N;  // 2 DT = KK products of V^T P^T, KK of S^T
    const int k_now = k_in((t + 1) & 1), v_now = v_in(out ? 2 : t & 1);
    const auto fetch = [&](int i) -> Frag { return i < KK ? vfrag(v_now, i / DT, i % DT) : kfrag(k_now, i - KK); };
    Frag ring[RING];
#pragma unroll
    for (int i = 0; i < RING; ++i) ring[i] = fetch(i);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const Frag f = ring[i % RING];
      if (i + RING < N) ring[i % RING] = fetch(i + RING);
      if (i < KK) {
#pragma unroll
        for (int n = 0; n < TERMS_P; ++n) acc[i % DT] = attn::Mma<E>::run(f, p[i / DT][n], acc[i % DT]);
      } else {
        if (i == KK) {
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = 0.f;
        }
#pragma unroll
        for (int n = 0; n < TERMS_Q; ++n) s = attn::Mma<E>::run(f, q[i - KK][n], s);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    stage.store_k(k1 - key0 - 2 * kTile, lds.k[t & 1]);
    stage.store_v(k1 - key0 - kTile, lds.v[(t + 1) & 1]);
    __syncthreads();
  }

  // The tiles left: their values one key at a time, added to the rows that see it. (Apart
  // from the loop above, whose registers this took when it was part of it.)
  if (__syncthreads_or(left)) {
    const float base = m == -INFINITY ? 0.f : m;
    for (int t = max(0, (min(limit_of(row0), k1) - k0) / kTile); t < steps; ++t) {
      const int key0 = k0 + t * kTile;
      lk = look(t);
      __builtin_amdgcn_s_waitcnt(0x0F70);
      stage.fetch_k(lk, 0, lds.k[0]);
      stage.fetch_v(lk, 0, lds.v[0]);
      stage.store_k(k1 - key0, lds.k[0]);
      stage.store_v(k1 - key0, lds.v[0]);
      __syncthreads();
      if (key0 + kTile > low && __any(wild_tile(lds.v[0]))) {
        s = scores(0);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const bool in = ((lk.there >> (r / 8)) & 1) && key0 + 8 * (r / 4) + 4 * g + r % 4 < limit;
          s[r] = in ? __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.c, -base)) : 0.f;
        }
#pragma unroll 1
        for (int key = 0; key < kTile; ++key) {
          // key 16 c + 8 (j / 4) + 4 g + j % 4 is element j of lane half g in product c
          const int c = key >> 4, j = 4 * ((key >> 3) & 1) + (key & 3);
          const bool mine = g == ((key >> 2) & 1);
          float e[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) e[i] = mine && i == j ? (c ? s[8 + i] : s[i]) : 0.f;
          w4 w[TERMS_P], mask;
          terms_of<E, TERMS_P>(e, w);
#pragma unroll
          for (int i = 0; i < 4; ++i) mask[i] = mine && i == j / 2 ? ((j & 1) ? 0xffff0000u : 0xffffu) : 0u;
          const bool in = key0 + key < limit;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            const Frag f = __builtin_bit_cast(Frag, __builtin_bit_cast(w4, vfrag(v_in(0), c, dt)) & mask);
            f32x16 add;
#pragma unroll
            for (int r = 0; r < 16; ++r) add[r] = 0.f;
#pragma unroll
            for (int n = 0; n < TERMS_P; ++n) add = attn::Mma<E>::run(f, __builtin_bit_cast(Frag, w[n]), add);
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[dt][r] += in ? add[r] : 0.f;
          }
        }
      }
      __syncthreads();
    }
  }

  l += __shfl_xor(l, 32, 64);
  const uint64_t any = __ballot(seen);
  const bool had = ((any >> r32) | (any >> (r32 + 32))) & 1;
  m = had ? fmaxf(m, -3.4028235e38f) : -INFINITY;
  const int row = 32 * wave + r32;  // in the block's tile
  if (row >= rows) return;
  const int64_t place = (((int64_t)x * a.kv_heads + h) * a.rows + row) * a.d;
  T* to = row_of<T>(a, it.s.start, h, row0 + row);
  if (joined && g == 0) {
    a.ml[place / a.d * 2] = m;
    a.ml[place / a.d * 2 + 1] = l;
  }
  const float inv = m == -INFINITY ? 0.f : 1.f / l;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int d = 32 * dt + 8 * b + 4 * g;
      const f32x4 v = {acc[dt][4 * b], acc[dt][4 * b + 1], acc[dt][4 * b + 2], acc[dt][4 * b + 3]};
      if (d < a.d) {
        if (joined) *reinterpret_cast<f32x4*>(a.part + place + d) = v;
        else store4(to + d, v * inv);
      }
    }
}

template <typename T, typename E, int DL, int TERMS_Q, int TERMS_P, class Stage>
int launch_wide(Args a, const Plan& p, hipStream_t s, const char* who) {
  set_plan(a, p);
  hipLaunchKernelGGL((attn_paged_wide_kernel<T, E, DL, TERMS_Q, TERMS_P, Stage>), dim3((unsigned)(p.items * a.kv_heads)),
                     dim3(kThreads), 0, s, a);
  launch_join<T>(a, p, s);
  return launched(who);
}

}  // namespace paged
}  // namespace pk
