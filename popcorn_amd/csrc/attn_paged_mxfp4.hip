// Attention over a paged cache held as MXFP4 (attn_paged.h).
#include "attn_paged.h"
#include "attn_paged_wide.h"

namespace pk {
namespace {

using namespace paged;

template <typename T, int DL> int launch_wide_mx(const Args& a, const Plan& p, hipStream_t s, const char* who) {
  constexpr int TERMS = sizeof(T) == 4 ? 3 : (__is_same(T, bf16) ? 1 : 2);
  return launch_wide<T, bf16, DL, TERMS, TERMS, StageMx<DL>>(a, p, s, who);
}

template <typename T> int launch_mx(const Args& a, const Plan& p, hipStream_t s, const char* who) {
  if (p.wide) {
    if constexpr (sizeof(T) == 4)
      return launch_wide_mx<T, 192>(a, p, s, who);  // nowhere else (plan_of)
    else
      return a.d <= 64    ? launch_wide_mx<T, 64>(a, p, s, who)
             : a.d <= 96  ? launch_wide_mx<T, 96>(a, p, s, who)
             : a.d <= 128 ? launch_wide_mx<T, 128>(a, p, s, who)
             : a.d <= 192 ? launch_wide_mx<T, 192>(a, p, s, who)
                          : launch_wide_mx<T, 256>(a, p, s, who);
  }
  return a.d <= 64    ? launch<RowsMx<T, 64>, 1, true>(a, p, s, who)
         : a.d <= 128 ? launch<RowsMx<T, 128>, 1, true>(a, p, s, who)
                      : launch<RowsMx<T, 256>, 1, true>(a, p, s, who);
}

}  // namespace
}  // namespace pk

extern "C" {

int pk_attn_paged_mxfp4(const void* q, const void* k_codes, const void* k_scales, const void* v_codes,
                        const void* v_scales, const int* block_table, const int* cache_lens, const int* cu_seqlens,
                        void* o, void* workspace, int64_t workspace_bytes, const int64_t* strides, int64_t num_seqs,
                        int64_t total, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t num_pages,
                        int64_t page_size, int64_t table_width, int64_t table_stride, float softmax_scale, int causal,
                        int dtype, void* stream) {
  using namespace pk;
  const char* who = "pk_attn_paged_mxfp4";
  paged::Args a{};
  a.q = q, a.k = k_codes, a.v = v_codes, a.o = o;
  a.ks = static_cast<const uint8_t*>(k_scales), a.vs = static_cast<const uint8_t*>(v_scales);
  a.table = block_table, a.lens = cache_lens, a.cu = cu_seqlens;
  paged::Plan p;
  bool empty;
  const int status = paged::paged_args(who, a, strides, num_seqs, total, q_heads, kv_heads, head_dim, num_pages, page_size,
                                       table_width, table_stride, softmax_scale, causal, dtype, true, workspace,
                                       workspace_bytes, p, &empty);
  if (status != PK_OK || empty) return status;
  // scales: (page, head, block) strides of k's and v's, after the eight strides of q and the codes
  const int64_t counts[3] = {num_pages, kv_heads, head_dim / 32};
  for (int i = 8; i < 14; ++i)
    if (counts[(i - 8) % 3] > 1 && (strides[i] < 0 || strides[i] % 4 != 0))
      return fail(PK_ERR_INVALID, "%s: stride %d = %lld is not a non-negative multiple of 4", who, i, (long long)strides[i]);
  if (((reinterpret_cast<uintptr_t>(k_scales) | reinterpret_cast<uintptr_t>(v_scales)) & 3u) != 0)
    return fail(PK_ERR_INVALID, "%s: the scales must be 4-byte aligned", who);
  for (int i = 8; i < 11; ++i)
    if (counts[i - 8] > 1 && strides[i] != strides[i + 3])
      return fail(PK_ERR_UNSUPPORTED, "%s: the keys' and the values' scales have different strides", who);
  if (head_dim > 32 && strides[10] * 8 > INT32_MAX)
    return fail(PK_ERR_UNSUPPORTED, "%s: the scales of a row span more than 2 GiB", who);
  a.spage = strides[8], a.shead = strides[9], a.sblock = head_dim > 32 ? (int)strides[10] : 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case PK_F32: return launch_mx<float>(a, p, s, who);
    case PK_BF16: return launch_mx<bf16>(a, p, s, who);
    default: return launch_mx<f16>(a, p, s, who);
  }
}

}  // extern "C"
