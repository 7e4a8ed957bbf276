// Host-side checks that the entry points of the 8-bit key/value cache share.
#pragma once

#include <cstdint>
#include <string>

#include "w4a16_kv.h"

namespace w4a16_internal {

void set_last_error(const std::string& message);   // w4a16_hip.hip: the message w4a16_last_error() returns

int kv_fail(int code, const std::string& message);
int check_kv_block(int64_t block, int code_type);
int check_kv_cache(const w4a16_kv_cache* cache);   // a batch of 0 has no pointers to check
int check_written(const w4a16_kv_cache& cache);    // refuses codes and scales that share memory with each other
int check_apart(const w4a16_kv_cache& read, const w4a16_kv_cache& written);   // `written` as check_written lets it be

// Whether a launch of so many workgroups is one that HIP takes (fewer than 2^32 threads).
inline bool launch_fits(__int128 workgroups, int threads) {
    return workgroups <= INT32_MAX && workgroups * threads <= UINT32_MAX;
}

}  // namespace w4a16_internal
