// What the library's other translation units see of a context (tapir_ctx itself belongs to engine.hip).
#pragma once
#include "../../include/tapir_hip.h"

namespace tapir {

struct CtxInfo {
  int device;   // HIP device of the context
  int dtype;    // TAPIR_F32 or TAPIR_BF16
  int n_cus;    // compute units (0 under the host emulator)
};

CtxInfo ctx_info(const tapir_ctx* c);
// records `msg` for tapir_last_error() and returns `code`; never throws
int ctx_fail(tapir_ctx* c, int code, const char* msg) noexcept;

}  // namespace tapir
