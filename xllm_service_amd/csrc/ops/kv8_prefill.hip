// Paged attention of prompt rows over a cache held in 8 bits (kv8.h), bf16 in and out,
// causal: the kernels of paged_rows.h over such pages.
//
// Weights are rounded to bf16, as over bf16 pages of 128-wide heads: 2^-8 of each at
// most, a thirty-second of what the values themselves were rounded by.
#include "paged_long.h"

namespace xllm {

static PagedRows kv8_rows(long tokens, int n_seqs, int G, int n_kv, int D,
                          int max_blocks) {
  return paged_rows_plan(tokens, n_seqs, G, n_kv, D, max_blocks, 1, false);
}
// floats of scratch that a call asks for
long kv8_prefill_scratch(long tokens, int n_seqs, int G, int n_kv, int D,
                         int max_blocks) {
  if (tokens == 0 || n_seqs <= 0) return 0;
  return kv8_rows(tokens, n_seqs, G, n_kv, D, max_blocks).scratch;
}

void launch_kv8_prefill(unsigned short* out, float* ws, const unsigned short* q,
                        const unsigned char* k_cache, const unsigned char* v_cache,
                        const float* kv_scale, const int* block_tables,
                        const int* cu_q, const int* seq_lens, long tokens,
                        int n_seqs, float scale, int n_qheads, int n_kv, int D,
                        int max_blocks, int n_blocks, long q_stride,
                        long out_stride, hipStream_t stream) {
  if (tokens == 0 || n_seqs <= 0) return;
  const PagedRows plan =
      kv8_rows(tokens, n_seqs, n_qheads / n_kv, n_kv, D, max_blocks);
  const Kv8Pages pages{reinterpret_cast<const float2*>(kv_scale), n_blocks};
  const auto* kc = reinterpret_cast<const unsigned short*>(k_cache);
  const auto* vc = reinterpret_cast<const unsigned short*>(v_cache);
  if (D == 128 && plan.least == 0 && !getenv("KV8_NOLONG") &&
      paged_long_takes(tokens, n_seqs, n_qheads / n_kv, n_kv, max_blocks)) {
    paged_long_of<true>(out, q, kc, vc, block_tables, cu_q, seq_lens, tokens, n_seqs,
                        scale, n_qheads, n_kv, max_blocks, q_stride, out_stride, pages,
                        stream);
    return;
  }
  auto go = D == 128 ? paged_rows_of<128, 1, false, true>
                     : paged_rows_of<64, 1, false, true>;
  go(out, ws, q, kc, vc, block_tables, cu_q, seq_lens, tokens, n_seqs, scale, n_qheads, n_kv, max_blocks, q_stride, out_stride, plan,
     PagedMore{}, PagedAhead{}, pages, stream);
}

}  // namespace xllm
