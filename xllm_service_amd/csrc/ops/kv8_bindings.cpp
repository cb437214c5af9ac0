// PyTorch bindings of the paged cache held in 8 bits (kv8.h): every check of arguments
// is here.
#include <hip/hip_runtime.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <torch/extension.h>

#include <tuple>

namespace xllm {
void launch_kv8_plan(int*, const int*, const int*, const int*, long*, long*, int*,
                     int*, int, int, long, int, int, hipStream_t);
void launch_kv8_write(unsigned char*, unsigned char*, float*, const unsigned short*,
                      const unsigned short*, const long*, int, int, int, long, long,
                      int, hipStream_t);
int kv8_decode_parts(int, int, int, int);
void launch_kv8_decode(unsigned short*, const unsigned short*, const unsigned char*,
                       const unsigned char*, const float*, const int*, const int*,
                       float*, float*, float, int, int, int, int, int, int, long,
                       long, hipStream_t);
long kv8_prefill_scratch(long, int, int, int, int, int);
void launch_kv8_prefill(unsigned short*, float*, const unsigned short*,
                        const unsigned char*, const unsigned char*, const float*,
                        const int*, const int*, const int*, long, int, float, int,
                        int, int, int, int, long, long, hipStream_t);
}  // namespace xllm

namespace {

using torch::Tensor;

hipStream_t stream_of(const Tensor& t) {
  return at::hip::getCurrentHIPStream(t.device().index()).stream();
}
unsigned char* bytes(const Tensor& t) {
  return static_cast<unsigned char*>(t.data_ptr());
}
unsigned short* words(const Tensor& t) {
  return static_cast<unsigned short*>(t.data_ptr());
}
// every row starts at a multiple of n bytes
bool on_bytes(const Tensor& t, int n) {
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % n == 0 &&
         (t.size(0) <= 1 || t.stride(0) * 2 % n == 0);
}

struct Cache { int blocks, n_kv, D; };
Cache check_cache(const Tensor& k, const Tensor& v, const Tensor& s) {
  for (auto* t : {&k, &v}) {
    TORCH_CHECK(t->is_cuda() && t->dtype() == torch::kFloat8_e4m3fn &&
                    t->is_contiguous(),
                "kv8: caches must be contiguous float8_e4m3fn on GPU");
    TORCH_CHECK(reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                "kv8: caches must begin on 16 bytes");
    TORCH_CHECK(t->device() == s.device(), "kv8: cache on several devices");
  }
  TORCH_CHECK(s.is_cuda() && s.dtype() == torch::kFloat && s.is_contiguous() &&
                  reinterpret_cast<uintptr_t>(s.data_ptr()) % 8 == 0,
              "kv8: kv_scale must be contiguous float32 on GPU, on 8 bytes");
  TORCH_CHECK(k.dim() == 5 && v.dim() == 4 && s.dim() == 3,
              "kv8: k_cache [blocks, n_kv, D/16, 16, 16], v_cache [blocks, n_kv, D, "
              "16], kv_scale [blocks, n_kv, 2]");
  const long D = v.size(2);
  TORCH_CHECK(D == 64 || D == 128, "kv8: head_dim 64 or 128, not ", D);
  TORCH_CHECK(k.size(0) == s.size(0) && v.size(0) == s.size(0) &&
                  k.size(1) == s.size(1) && v.size(1) == s.size(1) &&
                  k.size(2) == D / 16 && k.size(3) == 16 && k.size(4) == 16 &&
                  v.size(3) == 16 && s.size(2) == 2,
              "kv8: shapes of the cache do not match");
  TORCH_CHECK(s.size(0) > 0 && s.size(0) < (1L << 27) && s.size(1) > 0 &&
                  s.size(1) <= 4096,
              "kv8: a cache of 1 to 2^27 pages and of 1 to 4096 heads");
  return {(int)s.size(0), (int)s.size(1), (int)D};
}
// [T, heads, D] rows with packed heads
void check_rows(const Tensor& t, const Tensor& like, long D, const char* name) {
  TORCH_CHECK(t.device() == like.device() && t.dtype() == torch::kBFloat16,
              "kv8: ", name, " must be bf16 on the cache's device");
  TORCH_CHECK(t.dim() == 3 && t.size(2) == D, "kv8: ", name,
              " must be [tokens, heads, ", D, "]");
  TORCH_CHECK(t.stride(2) == 1 && (t.size(1) <= 1 || t.stride(1) == D) &&
                  (t.size(0) <= 1 || t.stride(0) >= 0),
              "kv8: heads of ", name, " must be packed");
  TORCH_CHECK(t.size(0) < (1L << 24), "kv8: too many rows");
}
void check_ints(const Tensor& t, const Tensor& like, int dims, const char* name) {
  TORCH_CHECK(t.device() == like.device() && t.dtype() == torch::kInt &&
                  t.is_contiguous() && t.dim() == dims,
              "kv8: ", name, " must be contiguous int32 of ", dims,
              " dimension(s) on the cache's device");
}

void write_pages(Tensor k, Tensor v, Tensor k_cache, Tensor v_cache, Tensor kv_scale,
           Tensor slots) {
  const Cache c = check_cache(k_cache, v_cache, kv_scale);
  const c10::DeviceGuard guard(kv_scale.device());
  check_rows(k, kv_scale, c.D, "k");
  check_rows(v, kv_scale, c.D, "v");
  TORCH_CHECK(k.size(1) == c.n_kv && v.size(1) == c.n_kv && k.size(0) == v.size(0),
              "kv8: k and v must have the cache's heads, and a row for each token");
  TORCH_CHECK(slots.device() == kv_scale.device() && slots.dtype() == torch::kLong &&
                  slots.is_contiguous() && slots.dim() == 1 &&
                  slots.size(0) == k.size(0),
              "kv8: slot_mapping must be contiguous int64, one for each token");
  if (k.size(0) == 0) return;
  // keys are read by 16 B, values by 4: copies of what lies at other addresses
  if (!on_bytes(k, 16)) k = k.clone(at::MemoryFormat::Contiguous);
  if (!on_bytes(v, 4)) v = v.clone(at::MemoryFormat::Contiguous);
  xllm::launch_kv8_write(bytes(k_cache), bytes(v_cache), kv_scale.data_ptr<float>(),
                         words(k), words(v), slots.data_ptr<long>(), (int)k.size(0),
                         c.n_kv, c.D, k.stride(0), v.stride(0), c.blocks,
                         stream_of(kv_scale));
}

// queries and results of attention
int check_attention(const Tensor& out, const Tensor& q, const Cache& c,
                    const Tensor& like) {
  check_rows(q, like, c.D, "q");
  check_rows(out, like, c.D, "out");
  TORCH_CHECK(out.sizes() == q.sizes() &&
                  (out.size(0) <= 1 || out.stride(0) >= out.size(1) * out.size(2)),
              "kv8: out must have the shape of q, and a place for each row");
  TORCH_CHECK(q.size(1) > 0 && q.size(1) % c.n_kv == 0,
              "kv8: query heads must be a multiple of the cache's");
  TORCH_CHECK(q.size(0) * q.size(1) < (1L << 27), "kv8: too many rows");
  return (int)(q.size(1) / c.n_kv);
}

// a launch has fewer than 2^32 threads
void check_grid(long n_seqs, const Cache& c) {
  TORCH_CHECK(n_seqs * c.n_kv < (1L << 22), "kv8: too many sequences");
}

// where results go: made here where the caller has none, 1 us less than by torch.empty
Tensor place_of(const c10::optional<Tensor>& out, const Tensor& q) {
  return out.has_value() ? *out : at::empty(q.sizes(), q.options());
}

Tensor attend_rows(Tensor q, Tensor k_cache, Tensor v_cache, Tensor kv_scale,
                   Tensor tables, Tensor lens, double scale,
                   c10::optional<Tensor> to) {
  const Cache c = check_cache(k_cache, v_cache, kv_scale);
  const c10::DeviceGuard guard(kv_scale.device());
  const Tensor out = place_of(to, q);
  const int G = check_attention(out, q, c, kv_scale);
  check_ints(tables, kv_scale, 2, "block_tables");
  check_ints(lens, kv_scale, 1, "seq_lens");
  const int S = q.size(0), H = q.size(1);
  TORCH_CHECK(G <= 16, "kv8: at most 16 query heads for each of the cache's");
  check_grid(S, c);
  TORCH_CHECK(tables.size(0) >= S && lens.size(0) >= S,
              "kv8: a table and a length for each sequence");
  TORCH_CHECK(tables.size(1) < (1L << 26), "kv8: tables too wide");
  if (S == 0) return out;
  if (!on_bytes(out, 8)) {                  // results are written by 8 B
    out.copy_(attend_rows(q, k_cache, v_cache, kv_scale, tables, lens, scale,
                          c10::nullopt));
    return out;
  }
  if (!on_bytes(q, 16)) q = q.clone(at::MemoryFormat::Contiguous);
  const int width = tables.size(1);
  const int parts = xllm::kv8_decode_parts(S, c.n_kv, G, width);
  Tensor ws;                                // parts, their sums, counters
  float *ws_o = nullptr, *ws_ml = nullptr;
  if (parts > 1) {
    const long n = (long)S * H * parts;
    ws = torch::empty({n * (c.D + 2) + 2L * S * c.n_kv},
                      kv_scale.options());
    ws_o = ws.data_ptr<float>();
    ws_ml = ws_o + n * c.D;
  }
  xllm::launch_kv8_decode(words(out), words(q), bytes(k_cache), bytes(v_cache),
                          kv_scale.data_ptr<float>(), tables.data_ptr<int>(),
                          lens.data_ptr<int>(), ws_ml, ws_o, (float)scale, S, H,
                          c.n_kv, c.D, width, c.blocks, q.stride(0), out.stride(0),
                          stream_of(kv_scale));
  return out;
}

Tensor attend_prompts(Tensor q, Tensor k_cache, Tensor v_cache, Tensor kv_scale,
                      Tensor tables, Tensor cu_q, Tensor lens, double scale,
                      c10::optional<Tensor> to) {
  const Cache c = check_cache(k_cache, v_cache, kv_scale);
  const c10::DeviceGuard guard(kv_scale.device());
  const Tensor out = place_of(to, q);
  const int G = check_attention(out, q, c, kv_scale);
  check_ints(tables, kv_scale, 2, "block_tables");
  check_ints(cu_q, kv_scale, 1, "cu_q");
  check_ints(lens, kv_scale, 1, "seq_lens");
  TORCH_CHECK(cu_q.size(0) > 0, "kv8: cu_q must have an entry more than sequences");
  check_grid(cu_q.size(0) - 1, c);
  const int S = cu_q.size(0) - 1, width = tables.size(1);
  TORCH_CHECK(tables.size(0) >= S && lens.size(0) >= S,
              "kv8: a table and a length for each sequence");
  TORCH_CHECK(tables.size(1) < (1L << 26), "kv8: tables too wide");
  const long T = q.size(0);
  if (T == 0 || S == 0) return out;
  if (!on_bytes(out, 8)) {                  // rows of no prompt stay as they are
    out.copy_(attend_prompts(q, k_cache, v_cache, kv_scale, tables, cu_q, lens, scale,
                             out.clone(at::MemoryFormat::Contiguous)));
    return out;
  }
  if (!on_bytes(q, 16)) q = q.clone(at::MemoryFormat::Contiguous);
  const long need = xllm::kv8_prefill_scratch(T, S, G, c.n_kv, c.D, width);
  Tensor ws;
  if (need > 0) ws = torch::empty({need}, kv_scale.options());
  xllm::launch_kv8_prefill(words(out), need > 0 ? ws.data_ptr<float>() : nullptr,
                           words(q), bytes(k_cache), bytes(v_cache),
                           kv_scale.data_ptr<float>(), tables.data_ptr<int>(),
                           cu_q.data_ptr<int>(), lens.data_ptr<int>(), T, S,
                           (float)scale, (int)q.size(1), c.n_kv, c.D, width,
                           c.blocks, q.stride(0), out.stride(0),
                           stream_of(kv_scale));
  return out;
}

std::tuple<Tensor, Tensor, Tensor, Tensor> plan_tables(Tensor tables, Tensor seq_lens,
                                                Tensor new_lens, Tensor free_blocks,
                                                long n_tokens) {
  TORCH_CHECK(tables.is_cuda() && tables.dtype() == torch::kInt && tables.dim() == 2 &&
                  (tables.size(1) <= 1 || tables.stride(1) == 1) &&
                  (tables.size(0) <= 1 || tables.stride(0) >= tables.size(1)),
              "block_tables must be int32 rows on GPU");
  const c10::DeviceGuard guard(tables.device());
  check_ints(seq_lens, tables, 1, "seq_lens");
  check_ints(new_lens, tables, 1, "new_lens");
  check_ints(free_blocks, tables, 1, "free_blocks");
  const long S = seq_lens.size(0);
  TORCH_CHECK(new_lens.size(0) == S && tables.size(0) >= S,
              "a new length and a table for each sequence");
  TORCH_CHECK(n_tokens >= 0 && n_tokens <= (1L << 20) && S < (1L << 24) &&
                  tables.size(1) < (1L << 26) && free_blocks.size(0) < (1L << 30),
              "too many tokens, sequences or pages");
  // one piece of memory for all four: an allocation takes 1.2 us
  const auto all = torch::empty({2 * n_tokens + (S + 3) / 2},
                                tables.options().dtype(torch::kLong));
  auto piece = [&](caffe2::TypeMeta type, long from, long n) {
    auto t = at::detail::make_tensor<c10::TensorImpl>(
        c10::Storage(all.storage()), all.key_set(), type);
    t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
    t.unsafeGetTensorImpl()->set_storage_offset(from);
    return t;
  };
  const auto longs = all.dtype(), ints = tables.dtype();
  auto slots = piece(longs, 0, n_tokens);
  auto positions = piece(longs, n_tokens, n_tokens);
  auto cu_q = piece(ints, 4 * n_tokens, S + 1);
  auto used = piece(ints, 4 * n_tokens + S + 1, 1);
  xllm::launch_kv8_plan(
      tables.data_ptr<int>(), seq_lens.data_ptr<int>(), new_lens.data_ptr<int>(),
      free_blocks.data_ptr<int>(), slots.data_ptr<long>(),
      positions.data_ptr<long>(), cu_q.data_ptr<int>(), used.data_ptr<int>(), (int)S,
      (int)tables.size(1), tables.stride(0), (int)free_blocks.size(0), (int)n_tokens,
      stream_of(tables));
  return {slots, positions, cu_q, used};
}

}  // namespace

void bind_kv8(pybind11::module& m) {
  m.def("extend_block_tables", &plan_tables);
  m.def("reshape_and_cache_kv8", &write_pages);
  m.def("paged_attn_decode_kv8", &attend_rows);
  m.def("paged_attn_prefill_kv8", &attend_prompts);
}
