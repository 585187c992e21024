// int8.hpp — a mounted int8 layer, as int8.hip makes it.  Internal to the library.
#pragma once

#include <stdint.h>

// Codes [out][pitch], zeros from `in` on to whole 64 bytes and more; scales and bias
// [out] (the bias zeros where none was given).
struct welvet_hip_int8 {
  int32_t in, out, act;
  int64_t pitch;
  int8_t *codes;
  float *scales, *bias;
};
