// Rotary embedding of new tokens' queries and keys, and their keys and values
// appended to a paged cache, in one launch:
//
//   y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin   (p = positions[t], rows of the tables)
//
// NeoX pairs (j, j + half) or GPT-J pairs (2j, 2j + 1), channels from 2 half on
// copied; q -> yq, k -> yk and the cache row of slots[t], v -> its cache row.
// fp32 arithmetic, one rounding per output. The cache has q's type, or holds MXFP4
// (mxfp4.h): there the 32 channels of a block are quantised from the rotation
// before any rounding, and what the codes stand for is returned as yk and yv.
//
// A thread owns eight channels of one token and goes over a group of heads with
// its table values in registers, so the tables are read once a group; a rotated
// NeoX chunk reads its partner's eight channels as well, from the cache lines its
// row's other threads read. The eight channels, and not eight pairs, because a
// block of 32 channels is then four neighbouring threads whatever `half` is: its
// largest value is two lane exchanges away.
//
// Bound by HBM: q, k and v in, yq, yk and two cache rows out. A few tokens are
// bound by the latency of one pass of loads, so the heads split over blocks until
// the grid has about eight blocks a CU. 16384 bf16 tokens of 32/8 heads of 128: 98.5 us,
// 4.5 TB/s; 8192 into MXFP4: 53 us, 4.1 TB/s; 32 tokens: 5.7 us, a launch and its loads.
// What is written is not read again here, and its stores bypass the caches (102.5 us without).
#include "api.h"
#include "common.h"
#include "mxfp4.h"

namespace pk {
namespace {

constexpr int kThreads = 256;

struct AppendArgs {
  const void* x[3];  // q, k, v
  void* y[3];        // yq, yk and, in 4 bits, yv
  void* rows[2];     // k and v cache rows, or their codes
  uint8_t* scales[2];
  const void* cos;
  const void* sin;
  const void* positions;
  const void* slots;
  int64_t xs[3][2];  // (token, head) strides
  int64_t rs[2][3];  // (page, head, token) strides of the cache rows or codes
  int64_t ss[2][3];  // (page, head, block) strides of the scales
  int64_t cache_rows, max_positions;
  int heads[3];
  int tokens, head_dim, half, page;
  int cs_dtype, wide_positions, wide_slots, interleaved;
  int chunks, rows_per_block, tiles, group;
};

// Eight consecutive elements at any element's address
template <typename T> struct alignas(16) Chunk {
  T v[8];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
      reinterpret_cast<u32x4*>(v)[i] = reinterpret_cast<const u32x4_any*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
      __builtin_nontemporal_store(reinterpret_cast<const u32x4*>(v)[i], reinterpret_cast<u32x4_any*>(p) + i);
  }
};

__device__ __forceinline__ float table_at(const void* p, int64_t i, int dtype) {
  if (dtype == kF32) return static_cast<const float*>(p)[i];
  return dtype == kBF16 ? to_f32(static_cast<const bf16*>(p)[i]) : to_f32(static_cast<const f16*>(p)[i]);
}

__device__ __forceinline__ int64_t index_at(const void* p, int64_t i, int wide) {
  return wide ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
}

// What a chunk of eight output channels is made of.
struct Turn {
  float c[8], s[8];  // y = x c + partner s, s negative in the first of a pair
  int partner[8];    // the partner's offset from the channel
  unsigned turned;   // channels that are rotated at all
};

// The sum of two exact products in 64 bits, as the fp32 that rounds to the same
// code: towards zero, the last bit set where something was cut off. A border
// between codes has two significant bits, so no value reaches or crosses one.
__device__ __forceinline__ float sticky(double y) {
  if (!(fabs(y) <= 3.4028234663852886e38)) return (float)y * INFINITY;  // past the largest fp32, Inf and NaN: not finite
  float r = (float)y;
  if (fabs((double)r) > fabs(y)) r = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, r) - 1u);
  if ((double)r != y) r = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, r) | 1u);
  return r;
}

// Largest of four neighbouring lanes
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  const uint32_t a = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true);  // lanes 1, 0, 3, 2
  v = v > a ? v : a;
  const uint32_t b = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true);  // lanes 2, 3, 0, 1
  return v > b ? v : b;
}

// WHOLE: a chunk is rotated as a whole or not at all, and with one partner chunk.
template <typename T, bool MX, bool WHOLE>
__global__ __launch_bounds__(kThreads) void rope_append_kernel(AppendArgs a) {
  constexpr int U = 4;  // heads whose loads are in flight together
  const int tile = (int)(blockIdx.x % (unsigned)a.tiles);
  const int h_begin = (int)(blockIdx.x / (unsigned)a.tiles) * a.group;
  const int all = a.heads[0] + a.heads[1] + a.heads[2];
  const int h_end = min(h_begin + a.group, all);
  const int per_tile = a.rows_per_block * a.chunks;
  for (int it = threadIdx.x; it < per_tile; it += kThreads) {
    const int r = it / a.chunks, c0 = (it - r * a.chunks) * 8;
    const int t = tile * a.rows_per_block + r;
    if (t >= a.tokens) break;  // four lanes of a block of 32 channels together: they share the token
    Turn u;
    u.turned = 0;
    if (c0 < 2 * a.half && h_begin < a.heads[0] + a.heads[1]) {
      const int64_t at = index_at(a.positions, t, a.wide_positions);
      const int64_t row = (at < 0 ? 0 : (at >= a.max_positions ? a.max_positions - 1 : at)) * a.half;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int ch = c0 + i;
        if (!WHOLE && ch >= 2 * a.half) break;
        const bool first = a.interleaved ? (i & 1) == 0 : ch < a.half;
        const int j = a.interleaved ? ch >> 1 : (first ? ch : ch - a.half);
        u.c[i] = table_at(a.cos, row + j, a.cs_dtype);
        const float s = table_at(a.sin, row + j, a.cs_dtype);
        u.s[i] = first ? -s : s;
        u.partner[i] = a.interleaved ? (first ? 1 : -1) : (first ? a.half : -a.half);
        u.turned |= 1u << i;
      }
    }
    const int64_t slot = index_at(a.slots, t, a.wide_slots);
    const bool held = slot >= 0 && slot < a.cache_rows;
    int64_t page = 0, off = 0;
    if (held) {
      if (slot <= INT32_MAX) {  // the shorter division
        page = (uint32_t)slot / (uint32_t)a.page;
        off = (uint32_t)slot - (uint32_t)page * (uint32_t)a.page;
      } else {
        page = slot / a.page;
        off = slot - page * a.page;
      }
    }
    for (int hh = h_begin; hh < h_end; hh += U) {
      Chunk<T> x[U], p[U];
#pragma unroll
      for (int n = 0; n < U; ++n) {
        const int g = hh + n;
        if (g >= h_end) break;
        const int kind = g < a.heads[0] ? 0 : (g < a.heads[0] + a.heads[1] ? 1 : 2);
        const int h = kind == 0 ? g : (kind == 1 ? g - a.heads[0] : g - a.heads[0] - a.heads[1]);
        const T* row = static_cast<const T*>(a.x[kind]) + t * a.xs[kind][0] + h * a.xs[kind][1] + c0;
        x[n].load(row);
        if constexpr (WHOLE) {
          if (kind < 2 && u.turned && !a.interleaved) p[n].load(row + u.partner[0]);
        } else if (kind < 2) {
#pragma unroll
          for (int i = 0; i < 8; ++i) p[n].v[i] = (u.turned >> i) & 1 ? row[i + u.partner[i]] : x[n].v[i];
        }
      }
#pragma unroll
      for (int n = 0; n < U; ++n) {
        const int g = hh + n;
        if (g >= h_end) break;
        const int kind = g < a.heads[0] ? 0 : (g < a.heads[0] + a.heads[1] ? 1 : 2);
        const int h = kind == 0 ? g : (kind == 1 ? g - a.heads[0] : g - a.heads[0] - a.heads[1]);
        if constexpr (WHOLE) {
          if (a.interleaved) {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[n].v[i] = x[n].v[i ^ 1];
          }
        }
        const unsigned turned = kind < 2 ? u.turned : 0u;
        const int64_t at = ((int64_t)t * a.heads[kind] + h) * a.head_dim + c0;
        if (!MX || kind == 0) {
          Chunk<T> y;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float v = to_f32(x[n].v[i]) * u.c[i] + to_f32(p[n].v[i]) * u.s[i];
            y.v[i] = (turned >> i) & 1 ? from_f32<T>(v) : x[n].v[i];
          }
          if (kind < 2) y.store(static_cast<T*>(a.y[kind]) + at);
          if (kind > 0 && held) {
            const int64_t* rs = a.rs[kind - 1];
            y.store(static_cast<T*>(a.rows[kind - 1]) + page * rs[0] + h * rs[1] + off * rs[2] + c0);
          }
        } else {
          float y[8];
          uint32_t top = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            y[i] = to_f32(x[n].v[i]);
            if ((turned >> i) & 1)
              y[i] = sticky((double)to_f32(x[n].v[i]) * (double)u.c[i] + (double)to_f32(p[n].v[i]) * (double)u.s[i]);
            const uint32_t m = __builtin_bit_cast(uint32_t, y[i]) & 0x7fffffffu;
            top = top > m ? top : m;
          }
          const uint32_t e = mx::scale_byte(quad_max(top));
          const uint32_t codes = mx::encode8(y, e);
          if (held) {
            const int64_t* rs = a.rs[kind - 1];
            const int64_t* ss = a.ss[kind - 1];
            *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.rows[kind - 1]) + page * rs[0] + h * rs[1] + off * rs[2] +
                                         c0 / 2) = codes;
            if (c0 % 32 == 0) a.scales[kind - 1][page * ss[0] + h * ss[1] + (c0 / 32) * ss[2] + off] = (uint8_t)e;
          }
          float z[8];
          mx::decode8(codes, mx::scale_of(e), z);
          Chunk<T> out;
#pragma unroll
          for (int i = 0; i < 8; ++i) out.v[i] = from_f32<T>(z[i]);
          out.store(static_cast<T*>(a.y[kind]) + at);
        }
      }
    }
  }
}

template <typename T, bool MX> int launch(AppendArgs a, hipStream_t s, const char* who) {
  a.chunks = a.head_dim / 8;
  a.rows_per_block = kThreads / a.chunks;  // head_dim is at most 256: at least eight tokens
  a.tiles = (a.tokens + a.rows_per_block - 1) / a.rows_per_block;
  const int all = a.heads[0] + a.heads[1] + a.heads[2];
  int64_t groups = (8 * (int64_t)cu_count() + a.tiles - 1) / a.tiles;
  groups = groups < 1 ? 1 : (groups > all ? all : groups);
  a.group = (int)((all + groups - 1) / groups);
  groups = (all + a.group - 1) / a.group;
  const int64_t blocks = groups * a.tiles;
  if (blocks > INT32_MAX) return fail(PK_ERR_UNSUPPORTED, "%s: %lld blocks exceed the grid", who, (long long)blocks);
  const bool whole = a.interleaved ? a.half % 4 == 0 : a.half % 8 == 0;
  if (whole)
    hipLaunchKernelGGL((rope_append_kernel<T, MX, true>), dim3((unsigned)blocks), dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL((rope_append_kernel<T, MX, false>), dim3((unsigned)blocks), dim3(kThreads), 0, s, a);
  return launched(who);
}

// Checks and fields that both entry points share; PK_OK with *empty set: nothing to do.
int append_args(const char* who, AppendArgs& a, const int64_t* strides, int64_t tokens, int64_t q_heads, int64_t kv_heads,
                int64_t head_dim, int64_t half, int64_t max_positions, int64_t num_pages, int64_t page_size, int dtype,
                int cs_dtype, int wide_positions, int wide_slots, int interleaved, bool mxfp4, bool* empty) {
  *empty = false;
  if (tokens < 0 || q_heads < 0 || kv_heads < 0 || num_pages < 0) return fail(PK_ERR_INVALID, "%s: negative size", who);
  if (!known_dtype(dtype) || !known_dtype(cs_dtype))
    return fail(PK_ERR_UNSUPPORTED, "%s: dtype codes %d (q, k, v) and %d (tables)", who, dtype, cs_dtype);
  const int unit = mxfp4 ? 32 : 8;
  if (head_dim <= 0 || head_dim > 256 || head_dim % unit != 0)
    return fail(PK_ERR_UNSUPPORTED, "%s: head_dim=%lld (a multiple of %d up to 256)", who, (long long)head_dim, unit);
  if (half < 1 || 2 * half > head_dim)
    return fail(PK_ERR_INVALID, "%s: half=%lld does not lie between 1 and head_dim/2", who, (long long)half);
  if (max_positions < 1) return fail(PK_ERR_INVALID, "%s: the tables have no row", who);
  if (page_size < 16 || page_size % 16 != 0 || page_size > (1 << 20))
    return fail(PK_ERR_UNSUPPORTED, "%s: page_size=%lld is not a multiple of 16 up to 2^20", who, (long long)page_size);
  if (tokens > (1 << 30) || q_heads > (1 << 20) || kv_heads > (1 << 20) || num_pages > INT32_MAX)
    return fail(PK_ERR_UNSUPPORTED, "%s: shape too large", who);
  if (tokens == 0 || q_heads + kv_heads == 0) {
    *empty = true;
    return PK_OK;
  }
  if (!strides || !a.cos || !a.sin || !a.positions || !a.slots || (q_heads && (!a.x[0] || !a.y[0])) ||
      (kv_heads && (!a.x[1] || !a.x[2] || !a.y[1] || (mxfp4 && !a.y[2]))))
    return fail(PK_ERR_INVALID, "%s: null pointer", who);
  const bool cached = kv_heads > 0 && num_pages > 0;
  for (int i = 0; cached && i < 2; ++i)
    if (!a.rows[i] || (mxfp4 && !a.scales[i])) return fail(PK_ERR_INVALID, "%s: null pointer", who);
  for (int i = 0; i < 3; ++i)
    for (int n = 0; n < 2; ++n) a.xs[i][n] = strides[2 * i + n];
  for (int i = 0; i < 2; ++i)
    for (int n = 0; n < 3; ++n) a.rs[i][n] = strides[6 + 3 * i + n];
  if (mxfp4) {
    for (int i = 0; i < 2; ++i) {
      for (int n = 0; n < 3; ++n) {
        a.ss[i][n] = strides[12 + 3 * i + n];
        const int64_t count = n == 0 ? num_pages : (n == 1 ? kv_heads : page_size);
        if (count > 1 && a.rs[i][n] % 4 != 0) return fail(PK_ERR_INVALID, "%s: a stride of the codes is not a multiple of 4", who);
      }
      if ((reinterpret_cast<uintptr_t>(a.rows[i]) & 3u) != 0)
        return fail(PK_ERR_INVALID, "%s: the codes are not 4-byte aligned", who);
    }
  }
  a.heads[0] = (int)q_heads;
  a.heads[1] = a.heads[2] = (int)kv_heads;
  a.tokens = (int)tokens;
  a.head_dim = (int)head_dim;
  a.half = (int)half;
  a.page = (int)page_size;
  a.cache_rows = num_pages * page_size;
  a.max_positions = max_positions;
  a.cs_dtype = cs_dtype;
  a.wide_positions = wide_positions;
  a.wide_slots = wide_slots;
  a.interleaved = interleaved;
  return PK_OK;
}

}  // namespace
}  // namespace pk

extern "C" {

int pk_rope_append(const void* q, const void* k, const void* v, const void* cos, const void* sin, const void* positions,
                   const void* slots, void* yq, void* yk, void* k_cache, void* v_cache, const int64_t* strides,
                   int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t half,
                   int64_t max_positions, int64_t num_pages, int64_t page_size, int dtype, int cs_dtype,
                   int wide_positions, int wide_slots, int interleaved, void* stream) {
  using namespace pk;
  const char* who = "pk_rope_append";
  AppendArgs a{};
  a.x[0] = q, a.x[1] = k, a.x[2] = v;
  a.y[0] = yq, a.y[1] = yk;
  a.rows[0] = k_cache, a.rows[1] = v_cache;
  a.cos = cos, a.sin = sin, a.positions = positions, a.slots = slots;
  bool empty;
  const int status = append_args(who, a, strides, tokens, q_heads, kv_heads, head_dim, half, max_positions, num_pages,
                                 page_size, dtype, cs_dtype, wide_positions, wide_slots, interleaved, false, &empty);
  if (status != PK_OK || empty) return status;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case PK_F32: return launch<float, false>(a, s, who);
    case PK_BF16: return launch<bf16, false>(a, s, who);
    default: return launch<f16, false>(a, s, who);
  }
}

int pk_rope_append_mxfp4(const void* q, const void* k, const void* v, const void* cos, const void* sin,
                         const void* positions, const void* slots, void* yq, void* yk, void* yv, void* k_codes,
                         void* k_scales, void* v_codes, void* v_scales, const int64_t* strides, int64_t tokens,
                         int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t half, int64_t max_positions,
                         int64_t num_pages, int64_t page_size, int dtype, int cs_dtype, int wide_positions,
                         int wide_slots, int interleaved, void* stream) {
  using namespace pk;
  const char* who = "pk_rope_append_mxfp4";
  AppendArgs a{};
  a.x[0] = q, a.x[1] = k, a.x[2] = v;
  a.y[0] = yq, a.y[1] = yk, a.y[2] = yv;
  a.rows[0] = k_codes, a.rows[1] = v_codes;
  a.scales[0] = static_cast<uint8_t*>(k_scales), a.scales[1] = static_cast<uint8_t*>(v_scales);
  a.cos = cos, a.sin = sin, a.positions = positions, a.slots = slots;
  bool empty;
  const int status = append_args(who, a, strides, tokens, q_heads, kv_heads, head_dim, half, max_positions, num_pages,
                                 page_size, dtype, cs_dtype, wide_positions, wide_slots, interleaved, true, &empty);
  if (status != PK_OK || empty) return status;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case PK_F32: return launch<float, true>(a, s, who);
    case PK_BF16: return launch<bf16, true>(a, s, who);
    default: return launch<f16, true>(a, s, who);
  }
}

}  // extern "C"
