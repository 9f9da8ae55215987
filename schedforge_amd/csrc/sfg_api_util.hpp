// sfg_api_util.hpp -- errors of the C ABI's entry points (sfg_api.hip holds the
// calling thread's last message, sfg_hip_last_error()).
#pragma once

namespace sfg {

// Keeps the message and returns the code.
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
// SFG_ERR_DEVICE with the runtime's message if the last launch failed.
int check_launch(const char* what);

}  // namespace sfg
