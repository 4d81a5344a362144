#include "../../include/drlvae.h"

extern "C" {

// DRL_SRC_HASH: sha256 (first 16 hex digits) over the library's sources, passed in by csrc/Makefile; bench.py
// and tests/test_abi.py compare it with the hash of the tree they run from, so a stale prebuilt library shows.
#ifndef DRL_SRC_HASH
#define DRL_SRC_HASH "unknown"
#endif
#define DRL_STR2(x) #x
#define DRL_STR(x) DRL_STR2(x)
const char* drl_version(void) { return "drlvae 0.3 (gfx950; abi " DRL_STR(DRL_ABI_REVISION) "; src " DRL_SRC_HASH ")"; }

}  // extern "C"
