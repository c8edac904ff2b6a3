// What the front end's functions share: the profiler range of a call, status
// and device-error checks, the current stream.
#pragma once

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <nvtx3/nvToolsExt.h>

#include <optional>
#include <sstream>
#include <string>

#include "yl_kvpath.h"
#include "yllang_kvpath.h"

namespace yllang {

// NVTX range over one front-end call, so a profiler timeline (nsys, or ncu's
// --nvtx range filters) shows which call launched which kernels; costs a
// function-pointer check when no tool is attached.
class Range {
 public:
  explicit Range(const char *name) { nvtxRangePushA(name); }
  ~Range() { nvtxRangePop(); }
  Range(const Range &) = delete;
  Range &operator=(const Range &) = delete;
};

inline void CheckStatus(int status, const char *what) {
  if (status != YL_OK) {
    std::ostringstream os;
    os << what << ": " << yl_status_string(status) << " (" << status << "): " << yl_last_error();
    throw PanicError(os.str());
  }
}

// Debug mode (see DeviceErrorChecksEnabled): a call given no device error
// word runs with a private one; Check() then waits for the stream and throws
// PanicError naming the bits the kernels raised.
class DeviceErrorScope {
 public:
  DeviceErrorScope(const torch::Device &device, uint32_t *given, const char *what) : m_word_(given), m_what_(what) {
    if (given == nullptr && DeviceErrorChecksEnabled()) {
      m_private_ = torch::zeros({1}, torch::TensorOptions().dtype(torch::kInt32).device(device));
      m_word_ = reinterpret_cast<uint32_t *>(m_private_.data_ptr<int32_t>());
    }
  }
  uint32_t *word() const { return m_word_; }
  void Check() const {
    if (!m_private_.defined()) return;
    const auto bits = static_cast<uint32_t>(m_private_.item<int32_t>());
    if (bits != 0) {
      std::ostringstream os;
      os << m_what_ << ": device error bits 0x" << std::hex << bits << std::dec << " (" << DeviceErrorNames(bits)
         << ")";
      throw PanicError(os.str());
    }
  }

 private:
  torch::Tensor m_private_;
  uint32_t *m_word_;
  const char *m_what_;
};

// A caller's device error word: a 4-byte tensor on the call's device.
inline uint32_t *ErrorWordOf(const std::optional<torch::Tensor> &w, const torch::Device &device, const char *what) {
  if (!w) return nullptr;
  RuntimeCheck(w->numel() >= 1 && w->element_size() == 4 && w->device() == device,
               std::string(what) + ": error_word must be a 4-byte tensor on the call's CUDA device");
  return static_cast<uint32_t *>(w->data_ptr());
}

inline cudaStream_t CurrentStream(const torch::Tensor &t) {
  return reinterpret_cast<cudaStream_t>(c10::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

inline void CheckSameDeviceDtype(const torch::Tensor &ref, std::initializer_list<const torch::Tensor *> ts,
                          const char *what) {
  RuntimeCheck(ref.is_cuda(), std::string(what) + ": tensors must be CUDA tensors");
  for (const auto *t : ts) {
    RuntimeCheck(t->device() == ref.device(), std::string(what) + ": tensors on different devices");
    RuntimeCheck(t->scalar_type() == ref.scalar_type(), std::string(what) + ": tensors of different dtypes");
  }
}

}  // namespace yllang
