// C-ABI plumbing shared by every entry point: a thread-local error string
// and launch-status checking.  No entry point allocates device memory.
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <type_traits>
#include <utility>

#include "locks_hip.h"

namespace locks {

static thread_local char g_err[512] = "";

void set_error(const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
}

int check_launch(const char* what) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        set_error("%s launch failed: %s", what, hipGetErrorString(e));
        return -2;
    }
    return 0;
}

}  // namespace locks

extern "C" const char* locks_last_error(void) { return locks::g_err; }

extern "C" int32_t locks_abi_version(void) { return LOCKS_ABI_VERSION; }

// ---- entries called with their arguments as one array of 8-byte words --------
namespace {

// An integer word that its argument's type does not hold is refused: cut to 32 bits
// it would be another, good-looking value.
template <typename T>
bool word_fits(uint64_t w) {
    if constexpr (std::is_integral_v<T>) return static_cast<int64_t>(w) == static_cast<int64_t>(static_cast<T>(w));
    else return true;
}

template <typename T>
T word_as(uint64_t w) {
    if constexpr (std::is_same_v<T, float>) {
        double d;
        memcpy(&d, &w, sizeof(d));
        return (float)d;
    } else if constexpr (std::is_pointer_v<T>) {
        return reinterpret_cast<T>(w);
    } else {
        static_assert(std::is_integral_v<T>, "an integer, a float or a pointer");
        return static_cast<T>(w);
    }
}
template <typename... A, size_t... I>
int32_t call_with(int32_t (*entry)(A...), const uint64_t* w, std::index_sequence<I...>) {
    const bool fits[] = {word_fits<A>(w[I])...};
    for (size_t i = 0; i < sizeof...(A); ++i)
        if (!fits[i]) {
            locks::set_error("locks_call: word %d is %lld, its argument has 32 bits", (int)i, (long long)w[i]);
            return -1;
        }
    return entry(word_as<A>(w[I])...);
}
template <typename... A>
int32_t call_with(int32_t (*entry)(A...), const uint64_t* w, int32_t n) {
    if (n != (int32_t)sizeof...(A)) {
        locks::set_error("locks_call: %d words for an entry of %d arguments", n, (int)sizeof...(A));
        return -1;
    }
    return call_with(entry, w, std::index_sequence_for<A...>{});
}

}  // namespace

extern "C" int32_t locks_call(int32_t entry, const uint64_t* words, int32_t n) {
    if (!words) {
        locks::set_error("locks_call: null words");
        return -1;
    }
    switch (entry) {
        case LOCKS_CALL_TABLES_STEP: return call_with(locks_tables_step, words, n);
        case LOCKS_CALL_TABLES_TRIM: return call_with(locks_tables_trim, words, n);
        case LOCKS_CALL_QKV_WRITE: return call_with(locks_qkv_write, words, n);
        case LOCKS_CALL_WINDOW_DECODE: return call_with(locks_window_decode, words, n);
        case LOCKS_CALL_WINDOW_PREFILL: return call_with(locks_window_prefill, words, n);
        case LOCKS_CALL_PREFIX_DECODE: return call_with(locks_prefix_decode, words, n);
        default: locks::set_error("locks_call: no entry %d", entry); return -1;
    }
}
