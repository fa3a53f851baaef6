// Torch entry point of the attention over cache pages.
#include "common.h"
#include "host_utils.h"
#include "paged_attention.h"
#include "paged_host.h"

namespace af3 {

void paged_attention(torch::Tensor q, torch::Tensor k_pages, torch::Tensor v_pages,
                     c10::optional<torch::Tensor> k_scales, c10::optional<torch::Tensor> v_scales,
                     torch::Tensor page_table, torch::Tensor seq_lens, torch::Tensor cu_q,
                     c10::optional<torch::Tensor> sinks, torch::Tensor out, int64_t hq, int64_t hkv,
                     int64_t window, double scale, int64_t max_q_len, int64_t max_seq_len) {
  using namespace paged;
  check_cuda_bf16(q, "q");
  check_cuda_bf16(out, "out");
  Args a;
  a.p = make_pool(k_pages, v_pages, k_scales, v_scales, 16);
  const auto dev = q.get_device();
  auto ints = [&](const torch::Tensor& t, const char* name) {
    AF3_CHECK(t.is_cuda() && t.get_device() == dev && t.scalar_type() == torch::kInt,
              std::string(name) + " must be int32 on q's device");
  };
  AF3_CHECK(k_pages.size(3) == kD, "paged attention is built for head_dim 64");
  AF3_CHECK(hkv > 0 && hq > 0 && hq % hkv == 0 && k_pages.size(2) == hkv,
            "k_pages must be [pages, page_size, Hkv, 64] with Hkv dividing Hq");
  AF3_CHECK(hq / hkv <= 128, "at most 128 query heads per KV head");
  AF3_CHECK(k_pages.get_device() == dev && out.get_device() == dev, "tensors on different devices");
  AF3_CHECK(q.dim() == 2 && q.size(1) == hq * kD && q.stride(1) == 1, "q must be [T, Hq * 64] with contiguous rows");
  AF3_CHECK(out.dim() == 2 && out.size(0) == q.size(0) && out.size(1) == hq * kD && out.stride(1) == 1,
            "out must be [T, Hq * 64] with contiguous rows");
  AF3_CHECK(reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0 && (q.stride(0) % 8 == 0 || q.size(0) <= 1) &&
                reinterpret_cast<uintptr_t>(out.data_ptr()) % 16 == 0 &&
                (out.stride(0) % 8 == 0 || out.size(0) <= 1),
            "q and out rows must be 16-byte aligned");
  ints(page_table, "page_table");
  ints(seq_lens, "seq_lens");
  ints(cu_q, "cu_q");
  AF3_CHECK(seq_lens.dim() == 1 && seq_lens.is_contiguous() && cu_q.dim() == 1 && cu_q.is_contiguous() &&
                cu_q.size(0) == seq_lens.size(0) + 1,
            "seq_lens must be [B] and cu_q [B + 1]");
  AF3_CHECK(page_table.dim() == 2 && page_table.size(0) == seq_lens.size(0) &&
                (page_table.stride(1) == 1 || page_table.size(1) <= 1),
            "page_table must be [B, max_pages] with contiguous rows");
  if (sinks.has_value())
    AF3_CHECK(sinks->is_cuda() && sinks->get_device() == dev && sinks->scalar_type() == torch::kFloat32 &&
                  sinks->numel() == hq && sinks->is_contiguous(),
              "sinks must be fp32 [Hq] on q's device");
  AF3_CHECK(window >= 0 && window < INT32_MAX, "window must not be negative");
  AF3_CHECK(scale > 0, "scale must be positive");
  AF3_CHECK(q.size(0) < (int64_t(1) << 30) && seq_lens.size(0) < 65536, "batch too large");
  const c10::cuda::CUDAGuard guard(q.device());
  if (q.size(0) == 0 || seq_lens.size(0) == 0) return;
  a.q = reinterpret_cast<const __nv_bfloat16*>(q.data_ptr());
  a.ld_q = q.stride(0);
  a.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  a.ld_out = out.stride(0);
  a.table = page_table.data_ptr<int>();
  a.ld_table = page_table.stride(0);
  a.max_pages = (int)page_table.size(1);
  a.lens = seq_lens.data_ptr<int>();
  a.cu = cu_q.data_ptr<int>();
  a.sinks = sinks.has_value() ? sinks->data_ptr<float>() : nullptr;
  a.B = (int)seq_lens.size(0);
  a.T = (int)q.size(0);
  a.hq = (int)hq;
  a.hkv = (int)hkv;
  a.group = (int)(hq / hkv);
  a.window = (int)std::min<int64_t>(window, int64_t(1) << 30);  // (differences of positions stay in 32 bits)
  a.scale_log2 = (float)scale * kLog2e;
  auto stream = at::cuda::getCurrentCUDAStream();
  max_q_len = std::max<int64_t>(max_q_len, 1);
  max_seq_len = std::max<int64_t>(max_seq_len, 1);
  if (a.group <= kFewRows && std::min<int64_t>(max_q_len, a.T) * a.group <= kFewTotal)
    launch_few(a, std::min<int64_t>(max_q_len, a.T), max_seq_len, stream);
  else
    launch_chunk(a, max_q_len, max_seq_len, stream);
}

}  // namespace af3
