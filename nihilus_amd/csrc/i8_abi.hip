// extern "C" surface of the calls on int8 matrices with a scale per row: argument checks, then the launch functions.
#include "../../include/nihilus_amd/i8_abi.h"
#include "abi_checks.h"
#include "i8_device.h"

#include <cmath>
#include <initializer_list>

namespace {

using nh::aligned16;
using nh::as_stream;
using nh::from_hip;
using nh::overlap;
using nh::require_device;

constexpr int64_t MAX_ROWS		= int64_t{ 1 } << 22; // a quantize launch has a workgroup of up to 512 threads to each
constexpr int64_t MAX_K			= 131008; // 128 * 128 * K stays below 2^31, K a multiple of 64
constexpr int64_t MAX_FRAGMENTS = int64_t{ 1 } << 25; // of a matrix: a tile launch has a thread to each 16 bytes
constexpr int64_t MAX_TILES		= int64_t{ 1 } << 22; // of 256 x 256 sums: workgroups of 512 threads (i8_form_for takes these tiles where smaller ones would be too many)

inline int64_t element(int type) {
	return type == NH_F32 ? 4 : 2;
}
inline int check_matrix(int64_t rows, int64_t k) {
	NH_REQUIRE(rows >= 0 && k > 0, NH_ERR_SHAPE);
	NH_REQUIRE(rows <= MAX_ROWS && k <= MAX_K && nh::i8_strips(rows) * nh::i8_steps(k) <= MAX_FRAGMENTS, NH_ERR_TOO_LARGE);
	return NH_OK;
}
inline int check_type(int type) {
	NH_REQUIRE(type == NH_F32 || type == NH_F16 || type == NH_BF16, NH_ERR_ARGUMENT);
	return NH_OK;
}
inline int check_product(int64_t M, int64_t N, int64_t K) {
	NH_TRY(check_matrix(M, K));
	NH_TRY(check_matrix(N, K));
	NH_REQUIRE((M + 255) / 256 * ((N + 255) / 256) <= MAX_TILES, NH_ERR_TOO_LARGE);
	return NH_OK;
}
inline bool aligned_as(const void* p, int type) {
	return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(element(type)) == 0;
}
// rows of an operand that is quantized
inline int check_rows(const void* x, int type, int64_t stride, int64_t rows, int64_t k) {
	NH_REQUIRE(stride >= k || rows <= 1, NH_ERR_SHAPE);
	NH_REQUIRE(stride <= (int64_t{ 1 } << 40), NH_ERR_TOO_LARGE);
	NH_REQUIRE(x, NH_ERR_NULL_POINTER);
	NH_REQUIRE(aligned_as(x, type), NH_ERR_ALIGNMENT);
	return NH_OK;
}
inline int check_eps(float eps) {
	NH_REQUIRE(eps >= 0.0f && std::isfinite(eps), NH_ERR_ARGUMENT);
	return NH_OK;
}
inline int check_workspace(const void* workspace, int64_t bytes, int64_t need) {
	NH_REQUIRE(workspace || need == 0, NH_ERR_NULL_POINTER);
	NH_REQUIRE(aligned16(workspace), NH_ERR_ALIGNMENT);
	NH_REQUIRE(bytes >= need, NH_ERR_ARGUMENT);
	return NH_OK;
}

// What a call writes has no byte in common with what it reads, nor with anything else that it writes.
struct part {
	const void* at;
	int64_t bytes;
};
inline int check_apart(std::initializer_list<part> written, std::initializer_list<part> read) {
	auto apart = [](const part& a, const part& b) {
		return a.bytes == 0 || b.bytes == 0 || !overlap(a.at, a.bytes, b.at, b.bytes);
	};
	for (const part* a = written.begin(); a != written.end(); ++a) {
		for (const part& b : read) {
			NH_REQUIRE(apart(*a, b), NH_ERR_ARGUMENT);
		}
		for (const part* b = written.begin(); b != a; ++b) {
			NH_REQUIRE(apart(*a, *b), NH_ERR_ARGUMENT);
		}
	}
	return NH_OK;
}
// rows of a stride
inline part rows_part(const void* x, int type, int64_t stride, int64_t rows, int64_t k) {
	return { x, ((rows - 1) * (rows > 1 ? stride : 0) + k) * element(type) };
}
inline part tiled_part(const void* p, int64_t rows, int64_t k) {
	return { p, nh::i8_bytes(rows, k) };
}
// y may be the residual
inline int check_result(const void* y, const void* residual, int64_t bytes) {
	return y == residual ? NH_OK : check_apart({ { y, bytes } }, { { residual, bytes } });
}

int quantize(const void* x, const void* up, const float* norm, float eps, int front, int type, int64_t stride, int64_t up_stride, void* tiled, int64_t rows, int64_t k, void* stream) {
	NH_TRY(check_type(type));
	NH_TRY(check_matrix(rows, k));
	NH_TRY(check_eps(eps));
	if (rows == 0) {
		return NH_OK;
	}
	NH_TRY(check_rows(x, type, stride, rows, k));
	if (front == nh::I8_SILU) {
		NH_TRY(check_rows(up, type, up_stride, rows, k));
	}
	NH_REQUIRE(tiled && (norm || front != nh::I8_NORM), NH_ERR_NULL_POINTER);
	NH_REQUIRE(aligned16(tiled) && aligned16(norm), NH_ERR_ALIGNMENT);
	NH_TRY(check_apart({ tiled_part(tiled, rows, k) }, { rows_part(x, type, stride, rows, k), rows_part(up, type, up_stride, rows, k), { norm, 4 * k } }));
	NH_TRY(require_device());
	nh::i8_rows in{};
	in.x = x, in.up = up, in.norm = norm, in.eps = eps;
	in.stride = rows > 1 ? stride : 0, in.up_stride = rows > 1 ? up_stride : 0;
	in.part = 1.0 / static_cast<double>(k);
	in.rows = static_cast<int>(rows), in.k = static_cast<int>(k);
	return from_hip(nh::launch_i8_quantize(in, front, type, tiled, as_stream(stream)));
}

} // namespace

extern "C" {

int64_t nh_i8_tiled_bytes(int64_t rows, int64_t k) {
	const int bad = check_matrix(rows, k);
	return bad ? bad : nh::i8_bytes(rows, k);
}

int nh_i8_quantize(const void* x, int type, int64_t x_stride, void* x_tiled, int64_t rows, int64_t k, void* stream) {
	return quantize(x, nullptr, nullptr, 0.0f, nh::I8_PLAIN, type, x_stride, 0, x_tiled, rows, k, stream);
}
int nh_i8_rms_norm_quantize(const void* x, int type, int64_t x_stride, const float* norm_weight, float eps, void* x_tiled, int64_t rows, int64_t k, void* stream) {
	return quantize(x, nullptr, norm_weight, eps, nh::I8_NORM, type, x_stride, 0, x_tiled, rows, k, stream);
}
int nh_i8_silu_mul_quantize(const void* gate, const void* up, int type, int64_t gate_stride, int64_t up_stride, void* x_tiled, int64_t rows, int64_t k, void* stream) {
	return quantize(gate, up, nullptr, 0.0f, nh::I8_SILU, type, gate_stride, up_stride, x_tiled, rows, k, stream);
}

static int check_tile(const void* tiled, const void* q, const void* scales, int64_t rows, int64_t k, bool to_tiled) {
	NH_TRY(check_matrix(rows, k));
	if (rows == 0) {
		return NH_OK;
	}
	NH_REQUIRE(tiled && q && scales, NH_ERR_NULL_POINTER);
	NH_REQUIRE(aligned16(tiled) && aligned_as(scales, NH_F32), NH_ERR_ALIGNMENT);
	const part t = tiled_part(tiled, rows, k), values{ q, rows * k }, steps{ scales, 4 * rows };
	NH_TRY(to_tiled ? check_apart({ t }, { values, steps }) : check_apart({ values, steps }, { t }));
	return require_device();
}
int nh_i8_tile(const int8_t* q, const float* scales, void* tiled, int64_t rows, int64_t k, void* stream) {
	NH_TRY(check_tile(tiled, q, scales, rows, k, true));
	return rows == 0 ? NH_OK : from_hip(nh::launch_i8_tile(q, scales, tiled, rows, k, as_stream(stream)));
}
int nh_i8_untile(const void* tiled, int8_t* q, float* scales, int64_t rows, int64_t k, void* stream) {
	NH_TRY(check_tile(tiled, q, scales, rows, k, false));
	return rows == 0 ? NH_OK : from_hip(nh::launch_i8_untile(tiled, q, scales, rows, k, as_stream(stream)));
}

int nh_i8_gemm(const void* w_tiled, const void* x_tiled, const void* residual, void* y, int type, int64_t M, int64_t N, int64_t K, void* stream) {
	NH_TRY(check_type(type));
	NH_TRY(check_product(M, N, K));
	if (M == 0 || N == 0) {
		return NH_OK;
	}
	NH_REQUIRE(w_tiled && x_tiled && y, NH_ERR_NULL_POINTER);
	NH_REQUIRE(aligned16(w_tiled) && aligned16(x_tiled) && aligned16(y) && aligned16(residual), NH_ERR_ALIGNMENT);
	NH_TRY(check_apart({ { y, M * N * element(type) } }, { tiled_part(w_tiled, N, K), tiled_part(x_tiled, M, K) }));
	NH_TRY(check_result(y, residual, M * N * element(type)));
	NH_TRY(require_device());
	return from_hip(nh::launch_i8_gemm(nh::i8_view(w_tiled, N, K), nh::i8_view(x_tiled, M, K), residual, y, type, as_stream(stream)));
}

int64_t nh_i8_mul_mat_workspace_bytes(int64_t M, int64_t K) {
	const int64_t bytes = nh_i8_tiled_bytes(M, K);
	return bytes > 0 && M == 1 && nh::i8_token_fits(1, 1, K, false) ? 0 : bytes; // (N and the norm are not known here)
}
int nh_i8_mul_mat(const void* w_tiled, const void* x, int type, int64_t x_stride, const float* norm_weight, float eps, const void* residual, void* y, int64_t M, int64_t N, int64_t K,
	void* workspace, int64_t workspace_bytes, void* stream) {
	NH_TRY(check_type(type));
	NH_TRY(check_product(M, N, K));
	NH_TRY(check_eps(eps));
	if (M == 0 || N == 0) {
		return NH_OK;
	}
	NH_TRY(check_rows(x, type, x_stride, M, K));
	NH_REQUIRE(w_tiled && y, NH_ERR_NULL_POINTER);
	NH_REQUIRE(aligned16(w_tiled) && aligned16(y) && aligned16(residual) && aligned16(norm_weight), NH_ERR_ALIGNMENT);
	NH_TRY(check_workspace(workspace, workspace_bytes, nh_i8_mul_mat_workspace_bytes(M, K)));
	const int64_t y_bytes = M * N * element(type);
	const part rows = rows_part(x, type, x_stride, M, K), norm{ norm_weight, 4 * K }, weights = tiled_part(w_tiled, N, K);
	NH_TRY(check_apart({ { y, y_bytes }, { workspace, nh_i8_mul_mat_workspace_bytes(M, K) } }, { rows, norm, weights }));
	NH_TRY(check_apart({ { workspace, nh_i8_mul_mat_workspace_bytes(M, K) } }, { { residual, y_bytes } }));
	NH_TRY(check_result(y, residual, y_bytes));
	if (nh::i8_token_fits(M, N, K, norm_weight != nullptr)) {
		NH_TRY(require_device());
		nh::i8_rows in{};
		in.x = x, in.norm = norm_weight, in.eps = eps, in.stride = x_stride;
		in.part = 1.0 / static_cast<double>(K);
		in.rows = static_cast<int>(M), in.k = static_cast<int>(K);
		return from_hip(nh::launch_i8_token(nh::i8_view(w_tiled, N, K), in, type, residual, y, as_stream(stream)));
	}
	NH_TRY(quantize(x, nullptr, norm_weight, eps, norm_weight ? nh::I8_NORM : nh::I8_PLAIN, type, x_stride, 0, workspace, M, K, stream));
	return nh_i8_gemm(w_tiled, workspace, residual, y, type, M, N, K, stream);
}

int64_t nh_i8_token_losses_workspace_bytes(int64_t M, int64_t N, int64_t K) {
	const int bad = check_product(M, N, K);
	return bad ? bad : M == 0 || N == 0 ? 0 : nh::i8_losses_workspace(M, N, K);
}
int nh_i8_token_losses(const void* w_tiled, const void* x_tiled, const int32_t* targets, float* losses, float* lse, int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes,
	void* stream) {
	NH_TRY(check_product(M, N, K));
	NH_REQUIRE(N > 0, NH_ERR_SHAPE);
	if (M == 0) {
		return NH_OK;
	}
	NH_REQUIRE(w_tiled && x_tiled && targets && losses && lse, NH_ERR_NULL_POINTER);
	NH_REQUIRE(aligned16(w_tiled) && aligned16(x_tiled) && aligned_as(targets, NH_F32) && aligned_as(losses, NH_F32) && aligned_as(lse, NH_F32), NH_ERR_ALIGNMENT);
	const int64_t need = nh_i8_token_losses_workspace_bytes(M, N, K);
	NH_TRY(check_workspace(workspace, workspace_bytes, need));
	NH_TRY(check_apart({ { losses, 4 * M }, { lse, 4 * M }, { workspace, need } }, { tiled_part(w_tiled, N, K), tiled_part(x_tiled, M, K), { targets, 4 * M } }));
	NH_TRY(require_device());
	return from_hip(nh::launch_i8_losses(nh::i8_view(w_tiled, N, K), nh::i8_view(x_tiled, M, K), { targets, losses, lse, static_cast<int>(K), workspace }, as_stream(stream)));
}

int64_t nh_i8_token_losses_grad_workspace_bytes(int64_t M, int64_t N, int64_t K, int type) {
	NH_TRY(check_type(type));
	const int bad = check_product(M, N, K);
	return bad ? bad : M == 0 || N == 0 ? 0 : nh::i8_gradient_workspace(M, N, K);
}
int nh_i8_token_losses_grad(const void* w_tiled, const void* x_tiled, const int32_t* targets, const float* losses, const float* lse, const float* grad, void* dx, int type, int64_t M, int64_t N,
	int64_t K, void* workspace, int64_t workspace_bytes, void* stream) {
	NH_TRY(check_type(type));
	NH_TRY(check_product(M, N, K));
	NH_REQUIRE(N > 0, NH_ERR_SHAPE);
	if (M == 0) {
		return NH_OK;
	}
	NH_REQUIRE(w_tiled && x_tiled && targets && losses && lse && dx, NH_ERR_NULL_POINTER);
	NH_REQUIRE(aligned16(w_tiled) && aligned16(x_tiled) && aligned16(dx), NH_ERR_ALIGNMENT);
	NH_REQUIRE(aligned_as(targets, NH_F32) && aligned_as(losses, NH_F32) && aligned_as(lse, NH_F32) && aligned_as(grad, NH_F32), NH_ERR_ALIGNMENT);
	const int64_t need = nh_i8_token_losses_grad_workspace_bytes(M, N, K, type);
	NH_TRY(check_workspace(workspace, workspace_bytes, need));
	NH_TRY(check_apart({ { dx, M * K * element(type) }, { workspace, need } },
		{ tiled_part(w_tiled, N, K), tiled_part(x_tiled, M, K), { targets, 4 * M }, { losses, 4 * M }, { lse, 4 * M }, { grad, 4 * M } }));
	NH_TRY(require_device());
	return from_hip(nh::launch_i8_gradient(nh::i8_view(w_tiled, N, K), nh::i8_view(x_tiled, M, K), { targets, losses, lse, grad, dx, static_cast<int>(K), type, workspace }, as_stream(stream)));
}

} // extern "C"
