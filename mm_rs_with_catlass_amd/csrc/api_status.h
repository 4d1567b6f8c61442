// What every entry point of the C ABI reports through (catcoc_last_error, catcoc_last_status, catcoc_last_launch).
#pragma once
#include "catcoc_hip.h"

namespace catcoc {

enum { E_NULL = 1, E_DESC = 2, E_SHAPE = 3, E_RANK = 4, E_TILING = 5, E_DTYPE = 6, E_WORKSPACE = 7, E_LAUNCH = 8 };

int api_fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));   // the calling thread's message and status; returns code
void api_launched(int hipError);                       // accepted, or what the launch itself answered
void api_launch_info(const CatcocLaunchInfo &info);    // what the call runs

}  // namespace catcoc
