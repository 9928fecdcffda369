// Error reporting of the C entry points (moegemm_last_error).
#pragma once

namespace moegemm {

// Keeps the formatted message for the calling thread and returns `code`.
int report(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

}  // namespace moegemm
