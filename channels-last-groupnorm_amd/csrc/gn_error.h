// The calling thread's error message (gnnhwc_last_error), set in gn_api.hip.
#pragma once
namespace gn {
// Formats the message and returns `code`.
int fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
}  // namespace gn
