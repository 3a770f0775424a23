// last_error.h -- the message behind pk_last_error(), for every source file of libparakeet_hip.so.
#pragma once

// Sets this thread's message (printf's format) and returns rc.
__attribute__((visibility("hidden"), format(printf, 2, 3))) int pk_fail(int rc, const char *fmt, ...);
// Clears it, as every entry point does first.
__attribute__((visibility("hidden"))) void pk_fail_clear();
