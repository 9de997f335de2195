// What the files of the C ABI share: argument checks, HIP's error codes as statuses, the device check.
#pragma once

#include "../../include/nihilus_amd/q8_0_abi.h"

#include <hip/hip_runtime.h>

#include <cstring>

namespace nh {

inline bool aligned16(const void* p) {
	return (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
}
// whether two pieces of memory (of at least a byte each) have one in common
inline bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
	const auto x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
	return a && b && x < y + static_cast<uintptr_t>(b_bytes) && y < x + static_cast<uintptr_t>(a_bytes);
}
inline hipStream_t as_stream(void* s) {
	return static_cast<hipStream_t>(s);
}
inline int from_hip(hipError_t e) {
	if (e == hipErrorNotReady) {
		return NH_ERR_BUSY; // the only source: the per-device scratch is still in use by a launch on another stream
	}
	return e == hipSuccess ? NH_OK : static_cast<int>(e);
}

// First call on a thread: make sure a gfx950 device is current.  Returns NH_OK or NH_ERR_NO_DEVICE.
inline int require_device() {
	static thread_local int cached = 1; // 1 = not checked yet
	if (cached != 1) {
		return cached;
	}
	int count = 0;
	if (hipGetDeviceCount(&count) != hipSuccess || count <= 0) {
		(void)hipGetLastError();
		return cached = NH_ERR_NO_DEVICE;
	}
	int dev = 0;
	hipDeviceProp_t prop;
	if (hipGetDevice(&dev) != hipSuccess || hipGetDeviceProperties(&prop, dev) != hipSuccess) {
		(void)hipGetLastError();
		return cached = NH_ERR_NO_DEVICE;
	}
	if (std::strncmp(prop.gcnArchName, "gfx950", 6) != 0) {
		return cached = NH_ERR_NO_DEVICE; // the code object holds gfx950 ISA only
	}
	return cached = NH_OK;
}

} // namespace nh

#define NH_REQUIRE(cond, code) \
	do {                       \
		if (!(cond)) {         \
			return (code);     \
		}                      \
	} while (0)
#define NH_TRY(expr)        \
	do {                    \
		const int rc_ = (expr); \
		if (rc_ != NH_OK) { \
			return rc_;     \
		}                   \
	} while (0)
