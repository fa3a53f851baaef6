// Host side of the page pools: argument checks and the device view.
#pragma once
#include "host_utils.h"
#include "paged.cuh"

namespace af3 {
namespace paged {

// `align`: bytes that every row of the pools has to be aligned to.
inline Pool make_pool(const torch::Tensor& k, const torch::Tensor& v,
                      const c10::optional<torch::Tensor>& ks, const c10::optional<torch::Tensor>& vs,
                      int64_t align) {
  AF3_CHECK(k.is_cuda() && v.is_cuda() && k.get_device() == v.get_device(),
            "pages must be CUDA tensors on one device");
  AF3_CHECK(k.dim() == 4 && k.sizes() == v.sizes(), "pages must be [pages, page_size, Hkv, D], K and V alike");
  AF3_CHECK(k.scalar_type() == v.scalar_type(), "K and V pages must have one type");
  AF3_CHECK(k.numel() > 0, "empty page pool");
  AF3_CHECK(k.strides() == v.strides() && k.stride(3) == 1,
            "K and V pages must have the same strides, rows contiguous");
  AF3_CHECK(k.size(0) < INT32_MAX && k.size(1) < (int64_t(1) << 24), "page pool too large");
  const bool fp8 = k.scalar_type() == at::kFloat8_e4m3fn;
  AF3_CHECK(fp8 || k.scalar_type() == torch::kBFloat16, "pages must be bfloat16 or float8_e4m3fn");
  const int64_t es = fp8 ? 1 : 2;
  Pool p;
  p.k = reinterpret_cast<uint8_t*>(k.data_ptr());
  p.v = reinterpret_cast<uint8_t*>(v.data_ptr());
  p.page = k.stride(0) * es;
  p.token = k.stride(1) * es;
  p.head = k.stride(2) * es;
  const bool aligned = reinterpret_cast<uintptr_t>(p.k) % align == 0 &&
                       reinterpret_cast<uintptr_t>(p.v) % align == 0 &&
                       (p.page % align == 0 || k.size(0) == 1) &&
                       (p.token % align == 0 || k.size(1) == 1) &&
                       (p.head % align == 0 || k.size(2) == 1);
  AF3_CHECK(aligned, "page rows must be " + std::to_string(align) + "-byte aligned");
  p.ks = p.vs = nullptr;
  p.s_page = p.s_head = p.s_token = 0;
  if (fp8) {
    AF3_CHECK(ks.has_value() && vs.has_value(), "float8_e4m3fn pages need k_scales and v_scales");
    AF3_CHECK(ks->is_cuda() && vs->is_cuda() && ks->get_device() == k.get_device() &&
                  vs->get_device() == k.get_device(),
              "scales must be on the pages' device");
    AF3_CHECK(ks->scalar_type() == torch::kUInt8 && vs->scalar_type() == torch::kUInt8,
              "scales must be uint8 (e8m0)");
    AF3_CHECK(ks->dim() == 3 && ks->size(0) == k.size(0) && ks->size(1) == k.size(2) &&
                  ks->size(2) == k.size(1) && ks->sizes() == vs->sizes() && ks->strides() == vs->strides(),
              "scales must be [pages, Hkv, page_size], K and V alike");
    p.ks = ks->data_ptr<uint8_t>();
    p.vs = vs->data_ptr<uint8_t>();
    p.s_page = ks->stride(0);
    p.s_head = ks->stride(1);
    p.s_token = ks->stride(2);
  } else {
    AF3_CHECK(!ks.has_value() && !vs.has_value(), "bfloat16 pages take no scales");
  }
  p.num_pages = (int)k.size(0);
  p.page_size = (int)k.size(1);
  p.page_shift = -1;
  for (int s = 0; s < 24; ++s)
    if ((1 << s) == p.page_size) p.page_shift = s;
  return p;
}

}  // namespace paged
}  // namespace af3
