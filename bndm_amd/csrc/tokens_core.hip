// Error reporting for libbndm_tokens.so.
#include "tokens_common.hpp"

namespace bndm {
static thread_local char g_tokens_err[512] = "";
void tokens_error(const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_tokens_err, sizeof(g_tokens_err), fmt, ap);
    va_end(ap);
}
}  // namespace bndm

extern "C" int bndm_tokens_abi_version(void) { return BNDM_TOKENS_ABI_VERSION; }
extern "C" const char *bndm_tokens_last_error(void) { return bndm::g_tokens_err; }
