// What the kernels on 8-bit rows with one scale each share: the layout of such a matrix, matrix instructions, the launch functions.
#pragma once

#include "../../include/nihilus_amd/i8_abi.h"
#include "q8_0_device.h"

namespace nh {

// A matrix [rows][k] of int8 with a scale per row: strips of 16 rows, in each strip steps of 64 values along k, each of them a fragment of 1 KiB in the order in which
// v_mfma_i32_16x16x64_i8 wants either operand: 16 bytes of lane l are row l % 16, values 16 (l / 16) .. + 15.  A fragment is fetched by one instruction of a wave, from memory or from LDS,
// where it lies as it came: no two lanes of an access meet in a bank.  Behind the strips, the scales of all (padded) rows.
constexpr int I8_ROWS	  = 16;
constexpr int I8_STEP	  = 64;
constexpr int I8_FRAGMENT = 1024;

inline __host__ __device__ int64_t i8_strips(int64_t rows) {
	return (rows + I8_ROWS - 1) / I8_ROWS;
}
inline __host__ __device__ int64_t i8_steps(int64_t k) {
	return (k + I8_STEP - 1) / I8_STEP;
}
inline int64_t i8_bytes(int64_t rows, int64_t k) {
	return i8_strips(rows) * (i8_steps(k) * I8_FRAGMENT + I8_ROWS * 4);
}

typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

struct i8_matrix {
	const v4u* q;
	const float* scale;
	int rows, strips, steps;
};
inline i8_matrix i8_view(const void* tiled, int64_t rows, int64_t k) {
	const int64_t strips = i8_strips(rows), steps = i8_steps(k);
	const char* p = static_cast<const char*>(tiled);
	return { reinterpret_cast<const v4u*>(p), reinterpret_cast<const float*>(p + strips * steps * I8_FRAGMENT), static_cast<int>(rows), static_cast<int>(strips), static_cast<int>(steps) };
}

// a value of type TYPE (NH_F32, NH_F16, NH_BF16) as fp32, and back with one rounding to nearest even
template<int TYPE> struct i8_type;
template<> struct i8_type<NH_F32> {
	typedef float store;
	static __device__ __forceinline__ float widen(float v) {
		return v;
	}
	static __device__ __forceinline__ float narrow(float v) {
		return v;
	}
};
template<> struct i8_type<NH_F16> {
	typedef uint16_t store;
	static __device__ __forceinline__ float widen(uint16_t v) {
		return half_bits_to_float(v);
	}
	static __device__ __forceinline__ uint16_t narrow(float v) {
		return float_to_half_bits(v);
	}
};
template<> struct i8_type<NH_BF16> {
	typedef uint16_t store;
	static __device__ __forceinline__ float widen(uint16_t v) {
		return __uint_as_float(static_cast<uint32_t>(v) << 16);
	}
	static __device__ __forceinline__ uint16_t narrow(float v) {
		return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v));
	}
};

// which rows are quantized
enum i8_front { I8_PLAIN, I8_NORM, I8_SILU };
struct i8_rows {
	const void* x;
	const void* up; // I8_SILU: x is the gate
	const float* norm; // I8_NORM
	int64_t stride, up_stride; // elements from one row to the next
	double part; // 1 / k
	float eps;
	int rows, k;
};

hipError_t launch_i8_quantize(const i8_rows& in, int front, int type, void* tiled, hipStream_t stream);
hipError_t launch_i8_tile(const int8_t* q, const float* scales, void* tiled, int64_t rows, int64_t k, hipStream_t stream);
hipError_t launch_i8_untile(const void* tiled, int8_t* q, float* scales, int64_t rows, int64_t k, hipStream_t stream);

// y [M][N] of `type` = x . w^T (+ residual), x [M][K], w [N][K]
hipError_t launch_i8_gemm(const i8_matrix& w, const i8_matrix& x, const void* residual, void* y, int type, hipStream_t stream);

// The same for a row, or a few, quantized in the launch: whether it is for these sizes, and it.
bool i8_token_fits(int64_t m, int64_t n, int64_t k, bool norm);
hipError_t launch_i8_token(const i8_matrix& w, const i8_rows& in, int type, const void* residual, void* y, hipStream_t stream);

struct i8_losses {
	const int32_t* targets;
	float *losses, *lse;
	int k;
	void* workspace;
};
int64_t i8_losses_workspace(int64_t m, int64_t n, int64_t k);
hipError_t launch_i8_losses(const i8_matrix& w, const i8_matrix& x, const i8_losses& l, hipStream_t stream);

struct i8_gradient {
	const int32_t* targets;
	const float *losses, *lse, *grad; // grad NULL: ones
	void* dx; // [M][k] of `type`
	int k, type;
	void* workspace;
};
int64_t i8_gradient_workspace(int64_t m, int64_t n, int64_t k);
hipError_t launch_i8_gradient(const i8_matrix& w, const i8_matrix& x, const i8_gradient& g, hipStream_t stream);

} // namespace nh
