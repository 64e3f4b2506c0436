// What the files of the torch operator layer share: status and device-error checks, the record of a nested tensor, dtype codes.
#pragma once

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <cstdlib>
#include <vector>

#include "ntb200.h"

namespace {

using at::Tensor;

[[maybe_unused]] void check_rc(int rc, const char* fn) {
  TORCH_CHECK(rc == NTB200_OK, "nestedtensor_b200: ", fn, " failed: ", ntb200_status_string(rc), " (", rc, ")");
}

// NTB200_CHECK_DEVICE_ERRORS=1: after every operator that runs a tcgen05 kernel, wait for the device and raise if one of
// its bounded waits ran out (the affected output tiles would otherwise be returned unwritten).  Off by default: the
// check synchronises.  Callers that leave it off poll nestedtensor_b200.device_error_flags() where it suits them.
[[maybe_unused]] void maybe_check_device_errors(const char* op) {
  static const bool enabled = [] {
    const char* v = std::getenv("NTB200_CHECK_DEVICE_ERRORS");
    return v != nullptr && v[0] != '\0' && v[0] != '0';
  }();
  if (!enabled) return;
  const int flags = ntb200_device_error_flags();
  TORCH_CHECK(flags == 0, "nestedtensor_b200: ", op, ": device error flags 0x", std::hex, flags,
              " (bits 0-2 projection, 8-10 attention, 12-14 attention backward: a bounded device-side wait ran out; bit 16: embedding index out of range)");
}

[[maybe_unused]] void* cur_stream() { return static_cast<void*>(at::cuda::getCurrentCUDAStream().stream()); }

struct Record {
  int64_t B;
  int64_t tdim;
  const int64_t* sz;  // host sizes, row stride tdim
  const int64_t* d_offsets;
  const int64_t* d_sizes;
  std::vector<int64_t> max_sizes;  // per tensor dim
  std::vector<bool> regular;       // per tensor dim: same extent in every constituent
  bool any_empty;
  int64_t numel;
};

[[maybe_unused]] Record make_record(const Tensor& sizes, const Tensor& meta) {
  TORCH_CHECK(sizes.device().is_cpu() && sizes.scalar_type() == at::kLong && sizes.dim() == 2 && sizes.is_contiguous(),
              "nestedtensor_b200: sizes must be a contiguous CPU int64 [B, tensor_dim] tensor");
  Record r;
  r.B = sizes.size(0);
  r.tdim = sizes.size(1);
  r.sz = sizes.data_ptr<int64_t>();
  TORCH_CHECK(meta.is_cuda(),
              "nestedtensor_b200: this operator needs a CUDA nested tensor (this build has no CPU implementation)");
  TORCH_CHECK(meta.scalar_type() == at::kLong && meta.is_contiguous() && meta.numel() == (r.B + 1) + r.B * r.tdim,
              "nestedtensor_b200: meta must be a CUDA int64 tensor of (B+1) + B*tensor_dim entries");
  r.d_offsets = meta.data_ptr<int64_t>();
  r.d_sizes = r.d_offsets + (r.B + 1);
  // One pass over the host sizes per operator call: kept branch-light (batches of 10^5 short sequences make this
  // loop, not the kernel, the cost of a call).
  constexpr int kMaxDims = 8;
  TORCH_CHECK(r.tdim <= kMaxDims, "nestedtensor_b200: at most ", kMaxDims, " tensor dimensions");
  int64_t mx[kMaxDims] = {0}, differs[kMaxDims] = {0}, min_seen = 0, numel = 0, empties = 0;
  const int64_t td = r.tdim;
  const int64_t* __restrict__ sz = r.sz;
  for (int64_t b = 0; b < r.B; ++b) {
    int64_t n = 1;
    for (int64_t j = 0; j < td; ++j) {
      const int64_t v = sz[b * td + j];
      min_seen = v < min_seen ? v : min_seen;
      n *= v;
      mx[j] = v > mx[j] ? v : mx[j];
      differs[j] |= v ^ sz[j];
    }
    empties += n == 0;
    numel += n;
  }
  TORCH_CHECK(min_seen >= 0, "nestedtensor_b200: negative size");
  r.max_sizes.assign(mx, mx + td);
  r.regular.resize(td);
  for (int64_t j = 0; j < td; ++j) r.regular[j] = differs[j] == 0;
  r.any_empty = empties != 0;
  r.numel = numel;
  return r;
}

[[maybe_unused]] void check_buffer(const Tensor& buffer, const Record& r, const char* op) {
  TORCH_CHECK(buffer.is_cuda(), "nestedtensor_b200: ", op,
              " needs a CUDA nested tensor (this build has no CPU implementation)");
  TORCH_CHECK(buffer.dim() == 1 && buffer.is_contiguous() && buffer.numel() == r.numel,
              "nestedtensor_b200: buffer must be 1-D contiguous with sum(numel) elements");
  const int64_t es = buffer.element_size();
  TORCH_CHECK(es == 1 || es == 2 || es == 4 || es == 8, "Input datatype ", buffer.dtype(), " is not supported.");
}

[[maybe_unused]] int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return NTB200_F32;
    case at::kHalf: return NTB200_F16;
    case at::kBFloat16: return NTB200_BF16;
    default: TORCH_CHECK(false, "nestedtensor_b200: this operator supports float32, float16 and bfloat16, got ", t);
  }
}

[[maybe_unused]] const void* opt_vec(const c10::optional<Tensor>& t, const Tensor& like, int64_t n, const char* name, Tensor* keep) {
  if (!t || !t->defined()) return nullptr;
  TORCH_CHECK(t->is_cuda() && t->device() == like.device() && t->scalar_type() == like.scalar_type(), "nestedtensor_b200: ",
              name, " must be on the input's device and of its dtype");
  TORCH_CHECK(t->numel() == n, "nestedtensor_b200: ", name, " must have ", n, " entries");
  *keep = t->contiguous();
  return keep->data_ptr();
}

}  // namespace
