// Attention over pages of fp8 codes (described in paged_attention.hip).
#include "paged_tiles.h"

int qkv::paged_call_fp8(const PagedCall& c, const char* what) { return paged_call<kFp8Pages>(c, what); }
