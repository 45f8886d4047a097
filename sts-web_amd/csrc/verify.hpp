// verify.hpp -- how far a draft holds against the target's probabilities.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace sts {

struct VerifyDraft {
  const float* target = nullptr;  // [B][T][V]
  const float* draft = nullptr;   // [B][T][V] or null
  const int32_t* tokens = nullptr;   // [B][T]
  const int32_t* parents = nullptr;  // [B][T]
  const int32_t* counts = nullptr;   // [B] or null: T
  const float* rand = nullptr;       // [B][T]
  int32_t* path = nullptr;           // [B][T]
  int32_t* accepted = nullptr;       // [B]
  int32_t* next = nullptr;           // [B]
  uint32_t T = 0, V = 0;
};
int launch_verify_draft(const VerifyDraft& p, uint32_t batch, hipStream_t stream);

}  // namespace sts
