// 8-bit products with a scale for each row of Y and each column of W:
//   out[i, j] = (sum_k q[i, k] * w[k, j]) * s[i] * t[j] (+ bias[j]),   q[i, k] = Y[i, k] / s[i] to the nearest whole number, s[i] = max |Y[i, :]| * (1 / 127)
// and the gated unit act(out of the first half of the columns) * (out of the second half), one kernel. The sums of 8-bit products are exact in 32 bits
// (at most 131,071 terms of 128 * 128), so an output carries the roundings of its scales' products and its own.
#include "../../include/cla_hip.h"
#include "k_q8.hpp"
#include "k_mm_out.hpp"
#include <algorithm>
#include <cmath>

namespace cla {

// ---- rows to 8 bits ----

template <class T> struct Q8Most { static __device__ __forceinline__ float value() { return 3.4028234663852886e38f; } };
template <> struct Q8Most<double> { static __device__ __forceinline__ double value() { return 1.7976931348623157e308; } };

// 8 neighbouring values of a row, `left` of them there (the others 0)
template <class T>
__device__ __forceinline__ void q8_load(const T* p, int64_t left, typename MmCalc<T>::type (&x)[8]) {
	typedef typename MmCalc<T>::type C;
	if(left >= 8) {
		T v[8];
		__builtin_memcpy(v, p, sizeof(v));
#pragma unroll
		for(int i = 0; i < 8; i++) x[i] = (C) v[i];
	}
	else {
#pragma unroll
		for(int i = 0; i < 8; i++) x[i] = i < left ? (C) p[i] : C(0);
	}
}

// Largest magnitude; infinity where a value is none (infinite or NaN).
template <class C>
__device__ __forceinline__ C q8_largest(const C (&x)[8], C m) {
#pragma unroll
	for(int i = 0; i < 8; i++) {
		const C a = fabs(x[i]);
		m = a <= Q8Most<C>::value() ? (a > m ? a : m) : (C) INFINITY;
	}
	return m;
}

// The scale of a row: the largest times 1 / 127, both in fp32. A row with a value that is not finite, or whose largest is none in fp32, has the scale NaN (and zeros): its outputs are NaN.
template <class C>
__device__ __forceinline__ float q8_scale(C largest) {
	const float a = (float) largest;
	return a <= 3.4028234663852886e38f ? a * (1.0f / 127.0f) : NAN;
}

// x / s to the nearest whole number, ties to even, as the exact quotient rounds. fp32: the product with the reciprocal is within one of it; x - r s is exact in
// fp32 next to s / 2 (both are multiples of half of s's last place, and below 2^24 of those), so comparing it with s / 2 decides. Scales whose reciprocal or
// last place leaves fp32's range take the fp64 quotient, whose distance from a half no fp32 operands can lose.
__device__ __forceinline__ int q8_round(float x, float s, float inv) {
	float r = rintf(x * inv);
	const float d = fmaf(-r, s, x), half = 0.5f * s;
	if(d > half || (d == half && ((int) r & 1))) r += 1.0f;
	else if(d < -half || (d == -half && ((int) r & 1))) r -= 1.0f;
	return (int) fminf(fmaxf(r, -127.0f), 127.0f);
}
__device__ __forceinline__ int q8_round_wide(double x, double s) { return (int) fmin(fmax(rint(x / s), -127.0), 127.0); }

template <class C>
__device__ __forceinline__ uint64_t q8_pack(const C (&x)[8], float s) {
	uint64_t v = 0;
	if(!(s > 0.0f)) return 0; // a row of zeros, or one with the scale NaN
	if(std::is_same<C, double>::value || s < 1e-30f) {
#pragma unroll
		for(int i = 0; i < 8; i++) v |= (uint64_t) (uint8_t) q8_round_wide((double) x[i], (double) s) << (8 * i);
	}
	else {
		const float inv = 1.0f / s;
#pragma unroll
		for(int i = 0; i < 8; i++) v |= (uint64_t) (uint8_t) q8_round((float) x[i], s, inv) << (8 * i);
	}
	return v;
}

// TPR threads to a row; what a thread holds of it (32 values) stays in registers between the search for the largest and the rounding, longer rows are read
// again. Bound: a row's bytes in and a quarter to a half of them out.
template <class T, int TPR>
__global__ __launch_bounds__(256) void k_q8_rows(const T* __restrict__ Y, int64_t m, int K, int64_t ld, int8_t* __restrict__ Q, int64_t ldQ, float* __restrict__ scale) {
	typedef typename MmCalc<T>::type C;
	constexpr int NV = 4;
	const int t = threadIdx.x % TPR;
	const int64_t row = (int64_t) blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
	if(TPR <= 64 && row >= m) return; // (TPR 256: the grid has m blocks)
	const T* const y = Y + row * ld;
	C x[NV][8], largest = C(0);
#pragma unroll
	for(int i = 0; i < NV; i++) {
		const int k = (i * TPR + t) * 8;
		q8_load<T>(y + k, K - k, x[i]);
		largest = q8_largest<C>(x[i], largest);
	}
	for(int k = (NV * TPR + t) * 8; k < K; k += TPR * 8) {
		C z[8];
		q8_load<T>(y + k, K - k, z);
		largest = q8_largest<C>(z, largest);
	}
#pragma unroll
	for(int d = (TPR < 64 ? TPR : 64) / 2; d > 0; d >>= 1) {
		const C o = __shfl_xor(largest, d, 64);
		largest = o > largest ? o : largest;
	}
	if(TPR > 64) {
		__shared__ C part[4];
		if((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = largest;
		__syncthreads();
#pragma unroll
		for(int i = 0; i < 4; i++) largest = part[i] > largest ? part[i] : largest;
	}
	const float s = q8_scale<C>(largest);
	if(t == 0) scale[row] = s;
	int8_t* const q = Q + row * ldQ;
	auto put = [&](int k, const C (&z)[8]) {
		const uint64_t v = q8_pack<C>(z, s);
		if(k + 8 <= K && (((uintptr_t) q | (uintptr_t) ldQ) & 7) == 0) *(uint64_t*) (q + k) = v;
		else
			for(int i = 0; i < 8 && k + i < K; i++) q[k + i] = (int8_t) (v >> (8 * i));
	};
#pragma unroll
	for(int i = 0; i < NV; i++) put((i * TPR + t) * 8, x[i]);
	for(int k = (NV * TPR + t) * 8; k < K; k += TPR * 8) {
		C z[8];
		q8_load<T>(y + k, K - k, z);
		put(k, z);
	}
}

template <class T>
static int q8_rows(const void* Y, int64_t m, int K, int64_t ld, int8_t* Q, int64_t ldQ, float* scale, hipStream_t stream) {
	if(m == 0) return 0;
	// up to 2048 values a wave holds a row in its registers (four rows to a block), beyond that a block does
	if(K <= 2048) k_q8_rows<T, 64><<<(unsigned) ((m + 3) / 4), 256, 0, stream>>>((const T*) Y, m, K, ld, Q, ldQ, scale);
	else k_q8_rows<T, 256><<<(unsigned) m, 256, 0, stream>>>((const T*) Y, m, K, ld, Q, ldQ, scale);
	CLA_HIP(hipGetLastError());
	return 0;
}

int launch_q8_rows(const void* Y, int type, int64_t m, int K, int64_t ld, int8_t* Q, int64_t ldQ, float* scale, hipStream_t stream) {
	switch(type) {
		case CLA_F64: return q8_rows<double>(Y, m, K, ld, Q, ldQ, scale, stream);
		case CLA_F32: return q8_rows<float>(Y, m, K, ld, Q, ldQ, scale, stream);
		case CLA_BF16: return q8_rows<__bf16>(Y, m, K, ld, Q, ldQ, scale, stream);
		default: return q8_rows<_Float16>(Y, m, K, ld, Q, ldQ, scale, stream);
	}
}

// ---- weights: a column's values one after the other, zeros up to a multiple of 128 ----

// byColumn: the source has a row per column already
__global__ __launch_bounds__(256) void k_q8_layout(const int8_t* __restrict__ src, int64_t ld, int byColumn, int64_t K, int N, int8_t* __restrict__ W, int64_t ldW) {
	__shared__ int8_t tile[64][65];
	const int64_t k0 = (int64_t) blockIdx.x * 64;
	const int n0 = blockIdx.y * 64;
	for(int i = threadIdx.x; i < 4096; i += 256) {
		const int a = i >> 6, b = i & 63;
		if(byColumn) tile[a][b] = n0 + a < N && k0 + b < K ? src[(int64_t) (n0 + a) * ld + k0 + b] : (int8_t) 0;
		else tile[b][a] = n0 + b < N && k0 + a < K ? src[(k0 + a) * ld + n0 + b] : (int8_t) 0;
	}
	__syncthreads();
	for(int i = threadIdx.x; i < 4096; i += 256) {
		const int a = i >> 6, b = i & 63;
		if(n0 + a < N) W[(int64_t) (n0 + a) * ldW + k0 + b] = tile[a][b]; // (ldW is a multiple of 128)
	}
}

int launch_q8_layout(const int8_t* src, int64_t ld, int byColumn, int64_t K, int N, int8_t* W, int64_t ldW, hipStream_t stream) {
	k_q8_layout<<<dim3((unsigned) (ldW / 64), (unsigned) ((N + 63) / 64)), 256, 0, stream>>>(src, ld, byColumn, K, N, W, ldW);
	CLA_HIP(hipGetLastError());
	return 0;
}

// Columns of a row-major matrix to rows of fp64, so that a column is quantised as a row is.
template <class T>
__global__ __launch_bounds__(256) void k_q8_columns(const T* __restrict__ src, int64_t ld, int64_t K, int N, double* __restrict__ dst) {
	__shared__ double tile[32][33];
	const int64_t k0 = (int64_t) blockIdx.x * 32;
	const int n0 = blockIdx.y * 32;
	for(int i = threadIdx.x; i < 1024; i += 256) {
		const int a = i >> 5, b = i & 31;
		if(k0 + a < K && n0 + b < N) tile[b][a] = (double) src[(k0 + a) * ld + n0 + b];
	}
	__syncthreads();
	for(int i = threadIdx.x; i < 1024; i += 256) {
		const int a = i >> 5, b = i & 31;
		if(n0 + a < N && k0 + b < K) dst[(int64_t) (n0 + a) * K + k0 + b] = tile[a][b];
	}
}

int launch_q8_columns(const void* src, int type, int64_t ld, int64_t K, int N, double* dst, hipStream_t stream) {
	const dim3 grid((unsigned) ((K + 31) / 32), (unsigned) ((N + 31) / 32));
	switch(type) {
		case CLA_F64: k_q8_columns<double><<<grid, 256, 0, stream>>>((const double*) src, ld, K, N, dst); break;
		case CLA_F32: k_q8_columns<float><<<grid, 256, 0, stream>>>((const float*) src, ld, K, N, dst); break;
		case CLA_BF16: k_q8_columns<__bf16><<<grid, 256, 0, stream>>>((const __bf16*) src, ld, K, N, dst); break;
		default: k_q8_columns<_Float16><<<grid, 256, 0, stream>>>((const _Float16*) src, ld, K, N, dst); break;
	}
	CLA_HIP(hipGetLastError());
	return 0;
}

// ---- products ----

template <class T> struct Q8Few {
	const int8_t* W;
	int64_t ldW;        // (a multiple of 128, zeros behind K)
	const float* t;
	const int8_t* Q;
	int64_t ldQ;
	const float* s;
	int32_t m, K, N, act;
	const T* bias;
	T* out;
	int64_t ld;
};

template <class T, bool GATED, int MR>
__global__ __launch_bounds__(64 * MMF_WAVES) void k_q8_few(Q8Few<T> A) {
	extern __shared__ __attribute__((aligned(16))) char q8_smem[]; // sums: [wave][half][row][column]
	typedef typename MmCalc<T>::type C;
	constexpr int H = GATED ? 2 : 1;
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n0 = blockIdx.x * 16;
	mm_i32x4 acc[H][MR];
	auto rowOf = [&](int row, int64_t k, int64_t) {
		return row < A.m && k < A.K ? *(const mm_i32x4*) (A.Q + row * A.ldQ + k) : mm_i32x4{0, 0, 0, 0};
	};
	mm_few<int8_t, GATED, MR>((const char*) A.W, A.ldW, n0, A.N, A.ldW, rowOf, acc, wave, lane);
	int* const red = (int*) q8_smem;
#pragma unroll
	for(int h = 0; h < H; h++)
#pragma unroll
		for(int j = 0; j < MR; j++)
			*(mm_i32x4*) (red + (((wave * H + h) * MR * 16) + 16 * j + (lane & 15)) * 16 + 4 * (lane >> 4)) = acc[h][j];
	__syncthreads();
	for(int i = threadIdx.x; i < A.m * 16; i += 64 * MMF_WAVES) {
		const int row = i >> 4, col = n0 + (i & 15);
		if(col >= A.N) continue;
		C x[H];
#pragma unroll
		for(int h = 0; h < H; h++) {
			int sum = 0;
#pragma unroll
			for(int w = 0; w < MMF_WAVES; w++) sum += red[(w * H + h) * MR * 256 + i];
			x[h] = (C) sum * ((C) A.s[row] * (C) A.t[col + h * A.N]);
			if(A.bias) x[h] += (C) A.bias[col + h * A.N];
		}
		A.out[row * A.ld + col] = (T) (GATED ? mm_act<T>(x[0], A.act) * x[H - 1] : x[0]);
	}
}

template <class T, bool GATED>
static int q8_few(const Q8Few<T>& A, hipStream_t stream) {
	const unsigned grid = (unsigned) ((A.N + 15) / 16);
	const int MR = A.m <= 16 ? 1 : A.m <= 32 ? 2 : 4;
	const size_t lds = (size_t) MMF_WAVES * (GATED ? 2 : 1) * MR * 1024;
	if(MR == 1) k_q8_few<T, GATED, 1><<<grid, 64 * MMF_WAVES, lds, stream>>>(A);
	else if(MR == 2) k_q8_few<T, GATED, 2><<<grid, 64 * MMF_WAVES, lds, stream>>>(A);
	else k_q8_few<T, GATED, 4><<<grid, 64 * MMF_WAVES, lds, stream>>>(A);
	CLA_HIP(hipGetLastError());
	return 0;
}

template <class T, bool GATED, int TM, int TN>
static int q8_tile(MmArgs A, const MmEpiOut<T, true>& epi, hipStream_t stream) {
	constexpr int WM = 2, WN = 2, NF = TN / WN / 32;
	constexpr size_t lds = std::max(2 * (TM + TN) * 128, WM * WN * MmEpiOut<T, true>::template region<int8_t, NF, GATED>());
	A.tilesM = (int32_t) ((A.M + TM - 1) / TM);
	A.tilesN = (A.N + (GATED ? TN / 2 : TN) - 1) / (GATED ? TN / 2 : TN);
	auto kernel = k_mm<int8_t, TM, TN, WM, WN, GATED, true, MmEpiOut<T, true>>;
	CLA_HIP(allow_full_lds((const void*) kernel));
	kernel<<<(unsigned) ((int64_t) A.tilesM * A.tilesN), 64 * WM * WN, lds, stream>>>(A, epi);
	CLA_HIP(hipGetLastError());
	return 0;
}

template <class T, bool GATED>
static int q8_mm(const Q8Product& p, hipStream_t stream) {
	const int N = GATED ? p.N / 2 : p.N; // columns of the output
	if(p.m <= Q8_FEW)
		return q8_few<T, GATED>(Q8Few<T>{p.W, p.ldW, p.t, p.Q, p.ldQ, p.s, (int32_t) p.m, p.K, N, p.act, (const T*) p.bias, (T*) p.out, p.ldOut}, stream);
	MmArgs A{};
	A.rows = (const char*) p.Q; A.ldRows = p.ldQ;
	A.cols = (const char*) p.W; A.ldCols = p.ldW;
	A.M = p.m; A.N = N; A.K = A.kPart = (p.K + 15) / 16 * 16; A.parts = 1;
	const MmEpiOut<T, true> epi{p.s, p.t, (const T*) p.bias, (T*) p.out, p.ldOut, p.act,
		(((uintptr_t) p.out | (uintptr_t) (p.ldOut * sizeof(T))) & 15) == 0, 0};
	const int64_t n = GATED ? 2 * (int64_t) N : N, big = ((p.m + 255) / 256) * ((n + 255) / 256), mid = ((p.m + 127) / 128) * ((n + 127) / 128);
	if(big >= g_numCU) return q8_tile<T, GATED, 256, 256>(A, epi, stream);
	if(mid >= g_numCU) return q8_tile<T, GATED, 128, 128>(A, epi, stream);
	return q8_tile<T, GATED, 64, 128>(A, epi, stream);
}

int launch_q8(const Q8Product& p, int type, bool gated, hipStream_t stream) {
	if(p.m == 0) return 0;
	switch(type) {
		case CLA_F64: return gated ? q8_mm<double, true>(p, stream) : q8_mm<double, false>(p, stream);
		case CLA_F32: return gated ? q8_mm<float, true>(p, stream) : q8_mm<float, false>(p, stream);
		case CLA_BF16: return gated ? q8_mm<__bf16, true>(p, stream) : q8_mm<__bf16, false>(p, stream);
		default: return gated ? q8_mm<_Float16, true>(p, stream) : q8_mm<_Float16, false>(p, stream);
	}
}

} // namespace cla
