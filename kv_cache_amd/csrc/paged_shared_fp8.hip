// Attention over shared prefixes in pages of fp8 codes (described in paged_shared.h).
#include "paged_shared.h"

int qkv::shared_call_fp8(const PagedCall& c, const int32_t* plan, const char* what) {
  return shared_call<kFp8Pages>(c, plan, what);
}
