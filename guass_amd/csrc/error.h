// error.h - the message that gf_last_error() returns, shared by the library's sources.
#ifndef GF_ERROR_H_
#define GF_ERROR_H_

// Stores `message` for this thread's gf_last_error() and returns `code` (a GF_E_* value).
__attribute__((visibility("hidden"))) int gf_set_error(int code, const char* message);

#endif  // GF_ERROR_H_
