// fa_status.h -- the device status: two words of device memory that kernels set
// once and the host reads (fa_device_status).  A wait that gave up and an index
// that was refused each have their own, so that neither hides the other.
#pragma once

namespace fa {

enum : int {
  STATUS_TIMEOUT = 0,  // (site << 8) | FA_ERR_DEVICE_TIMEOUT of the first wait that gave up
  STATUS_REFUSED = 1,  // (site << 8) | FA_ERR_BAD_INDEX of the first index out of range
  STATUS_WORDS = 2
};

// Both as one number: the timeout, or else the refused index, in bits 0..23
// (sites of waits go up to some hundreds); with both, the refused index's site,
// which is below 256, in bits 24..31.
inline int joined_status(const int* words) {
  const unsigned timeout = unsigned(words[STATUS_TIMEOUT]), refused = unsigned(words[STATUS_REFUSED]);
  return int(timeout ? timeout | (refused >> 8) << 24 : refused);
}

}  // namespace fa
