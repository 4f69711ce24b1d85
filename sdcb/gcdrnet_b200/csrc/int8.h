// int8.h -- what capi.cu needs of the int8 product (int8.cu).
#pragma once

namespace gcdr {

constexpr int GCDR_ERR_FLAG_OTHER = 1 << 30;   // the status itself could not be read

// Reads and clears the current device's error word of the int8 product (GCDR_ERR_FLAG_*).
int i8_status_word();

}  // namespace gcdr
