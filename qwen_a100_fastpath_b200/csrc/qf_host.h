// qf_host.h -- host helpers shared by the translation units of libqf_b200.
#pragma once
#include <string>

namespace qf {
// Records the message of a failing entry point (returned by qf_last_error_detail on this thread) and returns code.
int fail(int code, const std::string& msg);

// Checks that the current device is a B200 (sm_100a) and returns its index and SM count (either may be null).  The
// answer is kept per device; QF_OK or the code recorded by fail().
int require_b200(int* dev, int* sms);

// Reads and clears an `int` __device__ variable of the current device (synchronises the stream).
int read_error_word(const void* symbol, void* stream, int* status);
}  // namespace qf
