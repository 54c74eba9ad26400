// Attention over shared prefixes in pages of fp4 codes (described in paged_shared.h).
#include "paged_shared.h"

int qkv::shared_call_fp4(const PagedCall& c, const int32_t* plan, const char* what) {
  return shared_call<kFp4Pages>(c, plan, what);
}
