// Internal to the library: what aion_kv8.cu and aion_runtime.cu share.
#pragma once

#include "../../include/aion.h"

// Records the calling thread's last error text (aion_last_error(NULL)).
void aion_thread_error(const char* fmt, ...) __attribute__((format(printf, 1, 2)));
