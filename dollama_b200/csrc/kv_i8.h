// Shape and bookkeeping arrays of an int8 K/V cache call (kv_i8.cu).
#pragma once

namespace dlm {

struct KvShape {
  int B, S, H, Lmax;
  const int* pos;     // [B] position of each sequence's first new token
  const int* counts;  // [B] new tokens of each sequence, or null: S
  int* status;        // device status word
};

}  // namespace dlm
