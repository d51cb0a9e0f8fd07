// The message that tbk_last_error() returns, for every translation unit of the C ABI.
#pragma once

namespace tb {

// Keeps the formatted message for the calling thread and returns `code`.
int fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));

} // namespace tb
