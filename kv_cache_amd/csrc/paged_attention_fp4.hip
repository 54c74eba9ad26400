// Attention over pages of fp4 codes (described in paged_attention.hip).
#include "paged_tiles.h"

int qkv::paged_call_fp4(const PagedCall& c, const char* what) { return paged_call<kFp4Pages>(c, what); }
