// Identity of the serving operators' C ABI.
#include "pkda_common.h"
#include "serve/pkda_serve_gfx950.h"

extern "C" int pkda_serve_abi_version(void) { return PKDA_SERVE_ABI_VERSION; }

extern "C" int64_t pkda_serve_args_size(int which) {
  switch (which) {
    case PKDA_SERVE_ARGS_APPEND: return sizeof(pkda_paged_append_args);
    case PKDA_SERVE_ARGS_ATTENTION: return sizeof(pkda_paged_attention_args);
    case PKDA_SERVE_ARGS_SAMPLE: return sizeof(pkda_sample_args);
    default: return -1;
  }
}
