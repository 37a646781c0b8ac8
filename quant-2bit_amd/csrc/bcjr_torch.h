// Helpers of the torch operator sources: status check, current stream, device check.
#pragma once

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/library.h>

#include <optional>

#include "../../include/bcjr_hip.h"

namespace {

using at::Tensor;

// A failed C ABI call: a RuntimeError whose message starts with "bcjr status
// <n>:" (the Python package re-raises it as BcjrError with that status).
inline void check(int status, const char* what) {
  if (status != BCJR_OK)
    TORCH_CHECK(false, "bcjr status ", status, ": ", what, " failed: ", bcjr_strerror(status), ": ",
                bcjr_last_error());
}

inline hipStream_t stream_of(const Tensor& t) {
  return at::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

inline void same_device(const Tensor& ref, const std::optional<Tensor>& t, const char* name) {
  if (t) TORCH_CHECK(t->device() == ref.device(), name, " is on ", t->device(), " but the launch runs on ", ref.device());
}

}  // namespace
