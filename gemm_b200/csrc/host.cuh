// What the translation units of the library share on the host: the device's state, error words and
// the driver's tensor-map encoder (defined in launcher.cu).
#pragma once

#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <cstdint>

namespace neogemm {

// While one lives, the calling thread may allocate memory and load kernels although a stream is being
// captured: a process's first call may be made inside a capture.  Nothing that is done under it belongs
// to the captured work.
class RelaxedCapture {
 public:
  RelaxedCapture() { ok_ = cudaThreadExchangeStreamCaptureMode(&mode_) == cudaSuccess; }
  ~RelaxedCapture() {
    if (ok_) cudaThreadExchangeStreamCaptureMode(&mode_);
  }
  RelaxedCapture(const RelaxedCapture&) = delete;
  RelaxedCapture& operator=(const RelaxedCapture&) = delete;

 private:
  cudaStreamCaptureMode mode_ = cudaStreamCaptureModeRelaxed;
  bool ok_;
};

struct DeviceView {
  int index;          // CUDA device ordinal
  int sm_count;
  int* status;        // device address of the error word
  PFN_cuTensorMapEncodeTiled_v12000 encode;
};

// State of the current device, set up on first use.  Returns a neogemm_status code; an earlier
// launch's recorded error counts as one.
int acquire_device(DeviceView* out);

// Value of a tuning key on the calling thread (-1: default).
int tuning_value(int key);

// What neogemm_last_config() reports next on this thread.
void record_config(int cta_group, int columns, int stages, int swapped, int ctas, int tiles);

}  // namespace neogemm
