// Error plumbing of the libmme C ABI (include/mme.h).
//
// The reference reports failures as Python exceptions caught per model
// (main.py:822-824, 839-842); the ABI returns an int status and keeps the
// message in a thread-local buffer that the Python shim turns into RuntimeError.
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/mme.h"

static thread_local char g_err[512] = "";

int mme_set_error(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
    return code;
}

int mme_check_launch(const char* what) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return mme_set_error(MME_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
    return MME_OK;
}

// Exact, so that column ranges of one buffer pass: side by side at one leading dim by their distance within a row, at
// two leading dims row by row (of the block with fewer rows), which only blocks that reach into one another need.
bool mme_rows_overlap(const void* a, long lda, long ra, long wa, const void* b, long ldb, long rb, long wb) {
    typedef __int128 big;
    if (ra <= 0 || rb <= 0 || wa <= 0 || wb <= 0) return false;
    if (ra > rb) return mme_rows_overlap(b, ldb, rb, wb, a, lda, ra, wa);
    const big pa = (uintptr_t)a, pb = (uintptr_t)b, la = 2 * (big)lda, lb = 2 * (big)ldb, na = 2 * (big)wa, nb = 2 * (big)wb;
    if (pa + (ra - 1) * la + na <= pb || pb + (rb - 1) * lb + nb <= pa) return false;
    if (la == lb) {
        const big d = ((pb - pa) % la + la) % la;
        return d < na || la - d < nb;
    }
    for (long i = 0; i < ra; ++i) {
        const big x = pa + i * la - pb;                    // row i begins here, from b's begin
        const big j = x < nb ? 0 : (x - nb) / lb + 1;      // the first row of b that ends behind that
        if (j < rb && j * lb < x + na) return true;
    }
    return false;
}

extern "C" const char* mme_last_error(void) { return g_err; }
extern "C" int mme_abi_version(void) { return MME_ABI_VERSION; }
extern "C" int mme_build_flags(void) {
#ifdef MME_DEV
    return MME_BUILD_DEV;
#else
    return 0;
#endif
}
