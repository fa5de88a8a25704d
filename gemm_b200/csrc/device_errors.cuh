// Device-side error codes, written to the status word of a device (the first error wins).
#pragma once

namespace neogemm {

enum DeviceError : int {
  kDevOk = 0,
  kDevTimeoutProducer = 1,   // TMA warp gave up waiting for a free ring slot
  kDevTimeoutMmaFull = 2,    // MMA warp gave up waiting for operand bytes
  kDevTimeoutMmaTmem = 3,    // MMA warp gave up waiting for a drained accumulator
  kDevTimeoutEpilogue = 4,   // epilogue gave up waiting for a finished accumulator
  kDevTmemAddress = 5,       // tensor-memory allocation did not start at column 0 (pair mode)
  kDevBounds = 6,            // an index left its buffer (access skipped); aux: 1 partials,
                             // 2 counters, 3 C, 4 group offsets (clamped)
  kDevTimeoutScheduler = 7,  // a role gave up waiting on the dynamic-claim queue
};

}  // namespace neogemm
