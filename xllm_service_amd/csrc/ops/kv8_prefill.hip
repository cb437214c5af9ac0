// Paged attention of prompt rows over a cache held in 8 bits (kv8.h), bf16 in and out,
// causal: few rows by kv8_short.h, long prompts by paged_long.h, the rest by paged_rows.h.
//
// Weights are rounded to bf16, as over bf16 pages of 128-wide heads: 2^-8 of each at
// most, a sixteenth of what the values themselves were rounded by. What they are
// divided by is the sum of the rounded ones: made by products of pairs with ones, in half
// the additions, and exact results where one weight is all there is. (64-wide heads over
// bf16 pages have weights of three terms: who compares the two sees unequal work.)
//   kv8_short.h and paged_rows.h scale their sums only where a maximum has grown by more than
// 2^8: 3 to 8% of their time for errors of 0.0021 in place of 0.0018 of the results' size, of
// which rounding them to bf16 is 0.0016, and the values' rounding to 8 bits 0.02.
// paged_long.h, which would gain 1%, scales whenever one has grown.
#include "kv8_short.h"
#include "paged_long.h"

namespace xllm {

// Where kv8_short.h takes less time than paged_rows.h: one turn of its workgroups, two to
// a CU (three, 64 wide), and over long tables up to 1400 of them. A few of them over many
// keys go to the other kernel, which splits keys over workgroups, evenly those of a single
// sequence. 240 drawn batches, time over that of paged_rows.h: in one turn, up to so many
// keys, 0.40 to 1.18 (0.75), past them 0.76 to 2.1; more workgroups over enough keys 0.71 to
// 1.08 (0.90), over fewer 0.86 to 1.32. Us, paged_rows.h | here | bf16 pages: 300 tokens of
// 32/8 heads 15.0 | 9.8 | 12.8, 3 x 61-333 behind 0.5-3 k of 28/4 29.4 | 23.4 | 26.9, 100
// behind 800 28 | 11.7 | 14, 8 x 64-448 of 12/12 of 64 12.0 | 11.6 | 13.5.
static bool kv8_short_takes(long tokens, int n_seqs, int G, int n_kv, int D,
                            long max_blocks) {
  const long wgs = paged_rows_tiles<K8S_ROWS>(tokens, n_seqs, G) * n_kv;
  const long keys = max_blocks * PF_BS;
  if (wgs <= (D == 64 ? 768 : 512))
    return keys <= 1536 + (n_seqs == 1 ? 8 : 16) * wgs;
  return wgs <= 1400 && keys >= (D == 64 ? 700 : wgs <= 1024 ? 400 : 1000);
}

// Where paged_long.h takes less time: there a page is converted once for 256 rows, not
// 128, so earlier than with bf16 pages. By workgroups of 256 rows and the keys that a row
// sees on average, were the prompts equal. 170 drawn batches, time over that of
// paged_rows.h: from 440 workgroups on, over 550 keys 0.77 to 0.99 (0.88), 250 to 550 0.94
// to 1.09, fewer 1.02 to 1.17; 300 to 440, from 1200 keys on 0.79 to 0.96 (0.88), fewer 0.93
// to 1.17; 256 to 300, from 2500 on 0.85 to 1.05, fewer 0.98 to 1.30; below 1.0 to 1.4.
// Prompts of few rows leave most of 256 idle: 60 sequences of 160 rows over 2000 keys
// 0.72, 64 of 120 0.91, of 48 1.06, 128 of 16 1.18.
static bool kv8_long_takes(long tokens, int n_seqs, int G, int n_kv, int D,
                           long max_blocks) {
  if (D != 128 || tokens * G < 120L * n_seqs) return false;
  const long each = (tokens * G + n_seqs * (long)PL_ROWS - 1) / (n_seqs * (long)PL_ROWS);
  const long wgs = each * n_seqs * n_kv;
  const long sees = max_blocks * PF_BS - tokens / n_seqs / 2;
  return wgs >= 440 ? sees >= 550 : wgs >= 300 ? sees >= 1200 : wgs >= 256 && sees >= 2500;
}
static PagedRows kv8_rows(long tokens, int n_seqs, int G, int n_kv, int D,
                          int max_blocks) {
  return paged_rows_plan(tokens, n_seqs, G, n_kv, D, max_blocks, 1, false);
}
// floats of scratch that a call asks for
long kv8_prefill_scratch(long tokens, int n_seqs, int G, int n_kv, int D,
                         int max_blocks) {
  if (tokens == 0 || n_seqs <= 0 ||
      kv8_short_takes(tokens, n_seqs, G, n_kv, D, max_blocks) ||
      kv8_long_takes(tokens, n_seqs, G, n_kv, D, max_blocks))
    return 0;
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
  const Kv8Pages pages{reinterpret_cast<const float2*>(kv_scale), n_blocks};
  if (kv8_short_takes(tokens, n_seqs, n_qheads / n_kv, n_kv, D, max_blocks)) {
    auto go = D == 128 ? kv8_short<128> : kv8_short<64>;
    go(out, q, k_cache, v_cache, block_tables, cu_q, seq_lens, tokens, n_seqs, scale,
       n_qheads, n_kv, max_blocks, q_stride, out_stride, pages, stream);
    return;
  }
  const auto* kc = reinterpret_cast<const unsigned short*>(k_cache);
  const auto* vc = reinterpret_cast<const unsigned short*>(v_cache);
  if (kv8_long_takes(tokens, n_seqs, n_qheads / n_kv, n_kv, D, max_blocks)) {
    paged_long_of<true>(out, q, kc, vc, block_tables, cu_q, seq_lens, tokens, n_seqs,
                        scale, n_qheads, n_kv, max_blocks, q_stride, out_stride, pages,
                        stream);
    return;
  }
  const PagedRows plan =
      kv8_rows(tokens, n_seqs, n_qheads / n_kv, n_kv, D, max_blocks);
  auto go = D == 128 ? paged_rows_of<128, 1, false, true>
                     : paged_rows_of<64, 1, false, true>;
  go(out, ws, q, kc, vc, block_tables, cu_q, seq_lens, tokens, n_seqs, scale, n_qheads, n_kv, max_blocks, q_stride, out_stride, plan,
     PagedMore{}, PagedAhead{}, pages, stream);
}

}  // namespace xllm
