// Attention over a paged cache of q's type (attn_paged.h): the entry point and the
// workspace query of both caches.
#include "attn_paged.h"
#include "attn_paged_wide.h"

namespace pk {
namespace {

using namespace paged;

// fp32: both shapes on the kernel of few rows, 32 (16 at 256 dims) to a wave where they are many
template <int DL> int launch_rows32(const Args& a, const Plan& p, hipStream_t s, const char* who) {
  constexpr int R = DL <= 128 ? 2 : 1;
  return p.wide ? launch<Rows32<DL>, R, false>(a, p, s, who) : launch<Rows32<DL>, 1, true>(a, p, s, who);
}

template <typename T, int DL> int launch_wide16(const Args& a, const Plan& p, hipStream_t s, const char* who) {
  return launch_wide<T, T, DL, 1, 1, StageRows<T, DL>>(a, p, s, who);
}

template <typename T> int launch_rows(const Args& a, const Plan& p, hipStream_t s, const char* who) {
  if constexpr (sizeof(T) == 4)
    return a.d <= 64    ? launch_rows32<64>(a, p, s, who)
           : a.d <= 128 ? launch_rows32<128>(a, p, s, who)
                        : launch_rows32<256>(a, p, s, who);
  else if (p.wide)
    return a.d <= 64    ? launch_wide16<T, 64>(a, p, s, who)
           : a.d <= 96  ? launch_wide16<T, 96>(a, p, s, who)
           : a.d <= 128 ? launch_wide16<T, 128>(a, p, s, who)
           : a.d <= 192 ? launch_wide16<T, 192>(a, p, s, who)
                        : launch_wide16<T, 256>(a, p, s, who);
  else
    return a.d <= 64    ? launch<Rows16<T, 64>, 1, true>(a, p, s, who)
           : a.d <= 128 ? launch<Rows16<T, 128>, 1, true>(a, p, s, who)
                        : launch<Rows16<T, 256>, 1, true>(a, p, s, who);
}

}  // namespace
}  // namespace pk

extern "C" {

int64_t pk_attn_paged_workspace(int64_t num_seqs, int64_t total, int packed, int64_t q_heads, int64_t kv_heads,
                                int64_t head_dim, int64_t capacity, int dtype, int mxfp4) {
  using namespace pk;
  if (num_seqs < 0 || total < 0 || q_heads < 0 || kv_heads < 0 || head_dim < 0 || capacity < 0) return -1;
  if (total == 0 || q_heads == 0) return 0;
  if (kv_heads == 0 || q_heads % kv_heads != 0 || total * q_heads > INT32_MAX || num_seqs > (1 << 24)) return -1;
  const paged::Plan p = paged::plan_of(num_seqs, total, packed != 0, kv_heads, q_heads / kv_heads, head_dim, capacity,
                                        dtype == PK_F32, mxfp4 != 0);
  return p.part_bytes + p.ml_bytes + p.meta_bytes;
}

int pk_attn_paged(const void* q, const void* k_cache, const void* v_cache, const int* block_table, const int* cache_lens,
                  const int* cu_seqlens, void* o, void* workspace, int64_t workspace_bytes, const int64_t* strides,
                  int64_t num_seqs, int64_t total, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                  int64_t num_pages, int64_t page_size, int64_t table_width, int64_t table_stride, float softmax_scale,
                  int causal, int dtype, void* stream) {
  using namespace pk;
  const char* who = "pk_attn_paged";
  paged::Args a{};
  a.q = q, a.k = k_cache, a.v = v_cache, a.o = o;
  a.table = block_table, a.lens = cache_lens, a.cu = cu_seqlens;
  paged::Plan p;
  bool empty;
  const int status = paged::paged_args(who, a, strides, num_seqs, total, q_heads, kv_heads, head_dim, num_pages, page_size,
                                       table_width, table_stride, softmax_scale, causal, dtype, false, workspace,
                                       workspace_bytes, p, &empty);
  if (status != PK_OK || empty) return status;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case PK_F32: return launch_rows<float>(a, p, s, who);
    case PK_BF16: return launch_rows<bf16>(a, p, s, who);
    default: return launch_rows<f16>(a, p, s, who);
  }
}

}  // extern "C"
