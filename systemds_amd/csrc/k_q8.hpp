// 8-bit products: what their entry points ask of the kernels.
#pragma once
#include "cla_internal.hpp"

namespace cla {

constexpr int Q8_MAX_K = 131071;  // terms of a sum: 128 * 128 * 131,071 < 2^31
constexpr int Q8_MAX_N = 1 << 21; // columns: 65,536 blocks of 32 where they are laid out

struct Q8Product {
	const int8_t* W; int64_t ldW; const float* t;               // weights by column, their scales
	const int8_t* Q; int64_t ldQ; const float* s; int64_t m;    // rows, their scales
	int32_t K, N, act;
	const void* bias;
	void* out; int64_t ldOut;
	const void* Y; int64_t ldY;                                 // rows as they come, in place of Q and s (q8_fuses); null otherwise
};

// Whether the product quantises so few and short rows itself.
bool q8_fuses(int64_t m, int64_t K);

int launch_q8_rows(const void* Y, int type, int64_t m, int K, int64_t ld, int8_t* Q, int64_t ldQ, float* scale, hipStream_t stream);
int launch_q8_layout(const int8_t* src, int64_t ld, int byColumn, int64_t K, int N, int8_t* W, int64_t ldW, hipStream_t stream);
int launch_q8_columns(const void* src, int type, int64_t ld, int64_t K, int N, double* dst, hipStream_t stream);
int launch_q8(const Q8Product& p, int type, bool gated, hipStream_t stream);

} // namespace cla
