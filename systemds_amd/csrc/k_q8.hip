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

// 16 bytes of a row (V values), `left` values of them there (the others 0)
template <class T> struct Q8Piece {
	static constexpr int V = 16 / (int) sizeof(T);
	typedef typename MmCalc<T>::type C;
	static __device__ __forceinline__ mm_i32x4 load(const T* p, int64_t left) { return mm_load16<sizeof(T)>((const char*) p, left * (int) sizeof(T)); }
	static __device__ __forceinline__ C value(const mm_i32x4& p, int v) { return (C) __builtin_bit_cast(Vals, p).x[v]; }
	struct Vals { T x[V]; };
	// largest magnitude; infinity where a value is none (infinite or NaN)
	static __device__ __forceinline__ C largest(const mm_i32x4& p, C m) {
#pragma unroll
		for(int v = 0; v < V; v++) {
			const C a = fabs(value(p, v));
			m = a <= Q8Most<C>::value() ? (a > m ? a : m) : (C) INFINITY;
		}
		return m;
	}
};

// The scale of a row: the largest times 1 / 127, both in fp32. A row with a value that is not finite, or whose largest is none in fp32, has the scale NaN (and
// zeros): its outputs are NaN.
template <class C>
__device__ __forceinline__ float q8_scale(C largest) {
	const float a = (float) largest;
	return a <= 3.4028234663852886e38f ? a * (1.0f / 127.0f) : NAN;
}

// x / s to the nearest whole number, ties to even, as the exact quotient rounds: the product with the reciprocal is within one of it, and x - r s is exact next to
// s / 2 (both are multiples of x's or half of s's last place, below 2^24 or 2^53 of those), so comparing it with s / 2 decides. Scales whose reciprocal or
// last place leaves the range take the quotient in fp64, whose distance from a half no fp32 operands can lose.
template <class C>
__device__ __forceinline__ int q8_round(C x, C s, C inv) {
	C r = rint(x * inv);
	const C d = fma(-r, s, x), half = C(0.5) * s;
	const bool odd = ((int) r & 1) != 0;
	if(d > half || (d == half && odd)) r += C(1);
	else if(d < -half || (d == -half && odd)) r -= C(1);
	return (int) fmin(fmax(r, C(-127)), C(127));
}
template <class C>
__device__ __forceinline__ int q8_round_wide(C x, float s) { return (int) fmin(fmax(rint((double) x / (double) s), -127.0), 127.0); }

// TPR threads to a row, NV pieces each, which stay in registers between the search for the largest and the rounding; longer rows are read again. Bound: a
// row's bytes in and an eighth to a half of them out.
template <class T, int TPR, int NV>
__global__ __launch_bounds__(256) void k_q8_rows(const T* __restrict__ Y, int64_t m, int K, int64_t ld, int8_t* __restrict__ Q, int64_t ldQ, float* __restrict__ scale) {
	typedef Q8Piece<T> P;
	typedef typename P::C C;
	constexpr int V = P::V;
	const int t = threadIdx.x % TPR;
	const int64_t row = (int64_t) blockIdx.x * (256 / TPR) + threadIdx.x / TPR, at = min(row, m - 1); // (threads behind the last row follow it and write nothing)
	const T* const y = Y + at * ld;
	mm_i32x4 x[NV];
#pragma unroll
	for(int i = 0; i < NV; i++) x[i] = P::load(y + (i * TPR + t) * V, K - (i * TPR + t) * V);
	C largest = C(0);
#pragma unroll
	for(int i = 0; i < NV; i++) largest = P::largest(x[i], largest);
	for(int k = (NV * TPR + t) * V; k < K; k += TPR * V) largest = P::largest(P::load(y + k, K - k), largest);
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
	if(row >= m) return;
	const float s = q8_scale<C>(largest);
	if(t == 0) scale[row] = s;
	int8_t* const q = Q + row * ldQ;
	const bool whole = (((uintptr_t) Q | (uintptr_t) ldQ) & (V - 1)) == 0, none = !(s > 0.0f), wide = s < 1e-30f;
	const C inv = C(1) / (C) s;
	auto put = [&](int k, const mm_i32x4& p) {
		MmPack<int8_t, V> o;
#pragma unroll
		for(int v = 0; v < V; v++) o.x[v] = (int8_t) (none ? 0 : wide ? q8_round_wide<C>(P::value(p, v), s) : q8_round<C>(P::value(p, v), (C) s, inv));
		if(whole && k + V <= K) *(MmPack<int8_t, V>*) (q + k) = o;
		else {
#pragma unroll
			for(int v = 0; v < V; v++)
				if(k + v < K) q[k + v] = o.x[v];
		}
	};
#pragma unroll
	for(int i = 0; i < NV; i++)
		if(i * TPR * V < K) put((i * TPR + t) * V, x[i]);
	for(int k = (NV * TPR + t) * V; k < K; k += TPR * V) put(k, P::load(y + k, K - k));
}

template <class T>
static int q8_rows(const void* Yp, int64_t m, int K, int64_t ld, int8_t* Q, int64_t ldQ, float* scale, hipStream_t stream) {
	if(m == 0) return 0;
	constexpr int V = 16 / (int) sizeof(T);
	const T* const Y = (const T*) Yp;
	// Short rows 16 threads each, 16 rows a block; up to 8 pieces a lane a wave holds the row and no barrier is needed.
	const int64_t pieces = (K + V - 1) / V;
#define Q8_ROWS(TPR, NV) k_q8_rows<T, TPR, NV><<<(unsigned) ((m + 256 / TPR - 1) / (256 / TPR)), 256, 0, stream>>>(Y, m, K, ld, Q, ldQ, scale)
	if(pieces <= 16) Q8_ROWS(16, 1);
	else if(pieces <= 64) Q8_ROWS(16, 4);
	else if(m < 1024 || pieces > 64 * 8) {
		if(pieces <= 512) Q8_ROWS(256, 2);
		else Q8_ROWS(256, 8);
	}
	else if(pieces <= 64 * 2) Q8_ROWS(64, 2);
	else Q8_ROWS(64, 8);
#undef Q8_ROWS
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
	const T* Y;         // FUSE: rows as they come, in place of Q and s
	int64_t ldY;
};

// FUSE: each block quantises the rows itself, into LDS, while its first weights are on their way: up to Q8_FUSE rows that costs less than a kernel in front.
constexpr int Q8_FUSE = 4, Q8_FUSE_LDS = 64 << 10;

template <class T, bool GATED, int MR, bool FUSE>
__global__ __launch_bounds__(64 * MMF_WAVES) void k_q8_few(Q8Few<T> A) {
	extern __shared__ __attribute__((aligned(16))) char q8_smem[]; // sums: [wave][half][row][column]; FUSE: the 8-bit rows behind them
	typedef typename MmCalc<T>::type C;
	constexpr int H = GATED ? 2 : 1, SUMS = MMF_WAVES * H * MR * 1024;
	const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MR;
	if(!FUSE) { A.Q += m0 * A.ldQ; A.s += m0; }
	A.out += m0 * A.ld;
	A.m = min(A.m - m0, 16 * MR);
	__shared__ float scales[FUSE ? Q8_FUSE : 1];
	mm_i32x4 acc[H][MR];
	const int pitch = (A.K + 15) & ~15;
	auto quantise = [&]() {
		if constexpr(FUSE) {
			typedef Q8Piece<T> P;
			constexpr int V = P::V, NV = 2, NT = 64 * MMF_WAVES;
			__shared__ C part[Q8_FUSE][MMF_WAVES];
			mm_i32x4 x[Q8_FUSE][NV];
#pragma unroll
			for(int r = 0; r < Q8_FUSE; r++)
#pragma unroll
				for(int i = 0; i < NV; i++) x[r][i] = P::load(A.Y + min(r, A.m - 1) * A.ldY + (i * NT + tid) * V, r < A.m ? A.K - (i * NT + tid) * V : 0);
			C big[Q8_FUSE];
#pragma unroll
			for(int r = 0; r < Q8_FUSE; r++) {
				big[r] = C(0);
#pragma unroll
				for(int i = 0; i < NV; i++) big[r] = P::largest(x[r][i], big[r]);
				if(r < A.m)
					for(int k = (NV * NT + tid) * V; k < A.K; k += NT * V) big[r] = P::largest(P::load(A.Y + r * A.ldY + k, A.K - k), big[r]);
#pragma unroll
				for(int d = 32; d > 0; d >>= 1) {
					const C o = __shfl_xor(big[r], d, 64);
					big[r] = o > big[r] ? o : big[r];
				}
				if(lane == 0) part[r][wave] = big[r];
			}
			__syncthreads();
#pragma unroll
			for(int r = 0; r < Q8_FUSE; r++) {
				if(r >= A.m) break;
				C most = part[r][0];
#pragma unroll
				for(int w = 1; w < MMF_WAVES; w++) most = part[r][w] > most ? part[r][w] : most;
				const float s = q8_scale<C>(most);
				if(tid == 0) scales[r] = s;
				const bool none = !(s > 0.0f), wide = s < 1e-30f;
				const C inv = C(1) / (C) s;
				auto put = [&](int k, const mm_i32x4& p) { // (what lies behind the row is 0: so are the piece's bytes)
					MmPack<int8_t, V> o;
#pragma unroll
					for(int v = 0; v < V; v++) o.x[v] = (int8_t) (none ? 0 : wide ? q8_round_wide<C>(P::value(p, v), s) : q8_round<C>(P::value(p, v), (C) s, inv));
					*(MmPack<int8_t, V>*) (q8_smem + SUMS + r * pitch + k) = o;
				};
#pragma unroll
				for(int i = 0; i < NV; i++)
					if((i * NT + tid) * V < pitch) put((i * NT + tid) * V, x[r][i]);
				for(int k = (NV * NT + tid) * V; k < pitch; k += NT * V) put(k, P::load(A.Y + r * A.ldY + k, A.K - k));
			}
			__syncthreads();
		}
	};
	auto rowOf = [&](int row, int64_t k, int64_t) {
		const bool in = row < A.m && k < A.K;
		if(FUSE) return in ? *(const mm_i32x4*) (q8_smem + SUMS + row * pitch + k) : mm_i32x4{0, 0, 0, 0};
		return in ? *(const mm_i32x4*) (A.Q + row * A.ldQ + k) : mm_i32x4{0, 0, 0, 0};
	};
	mm_few<int8_t, GATED, MR>((const char*) A.W, A.ldW, n0, A.N, A.ldW, rowOf, quantise, acc, wave, lane);
	int* const red = (int*) q8_smem;
#pragma unroll
	for(int h = 0; h < H; h++)
#pragma unroll
		for(int j = 0; j < MR; j++)
			*(mm_i32x4*) (red + (((wave * H + h) * MR * 16) + 16 * j + (lane & 15)) * 16 + 4 * (lane >> 4)) = acc[h][j];
	__syncthreads();
	for(int i = tid; i < A.m * 16; i += 64 * MMF_WAVES) {
		const int row = i >> 4, col = n0 + (i & 15);
		if(col >= A.N) continue;
		const float s = FUSE ? scales[FUSE ? row : 0] : A.s[row];
		C x[H];
#pragma unroll
		for(int h = 0; h < H; h++) {
			int sum = 0;
#pragma unroll
			for(int w = 0; w < MMF_WAVES; w++) sum += red[(w * H + h) * MR * 256 + i];
			x[h] = (C) sum * ((C) s * (C) A.t[col + h * A.N]);
			if(A.bias) x[h] += (C) A.bias[col + h * A.N];
		}
		A.out[row * A.ld + col] = (T) (GATED ? mm_act<T>(x[0], A.act) * x[H - 1] : x[0]);
	}
}

template <class T, bool GATED>
static int q8_few(const Q8Few<T>& A, hipStream_t stream) {
	const int MR = A.Y ? 1 : mm_few_rows(A.m, A.N, g_numCU);
	const dim3 grid((unsigned) ((A.N + 15) / 16), (unsigned) ((A.m + 16 * MR - 1) / (16 * MR)));
	size_t lds = (size_t) MMF_WAVES * (GATED ? 2 : 1) * MR * 1024;
	if(A.Y) {
		lds += (size_t) A.m * ((A.K + 15) & ~15);
		CLA_HIP(allow_full_lds((const void*) k_q8_few<T, GATED, 1, true>));
		k_q8_few<T, GATED, 1, true><<<grid, 64 * MMF_WAVES, lds, stream>>>(A);
	}
	else if(MR == 1) k_q8_few<T, GATED, 1, false><<<grid, 64 * MMF_WAVES, lds, stream>>>(A);
	else if(MR == 2) k_q8_few<T, GATED, 2, false><<<grid, 64 * MMF_WAVES, lds, stream>>>(A);
	else {
		CLA_HIP(allow_full_lds((const void*) k_q8_few<T, GATED, 4, false>));
		k_q8_few<T, GATED, 4, false><<<grid, 64 * MMF_WAVES, lds, stream>>>(A);
	}
	CLA_HIP(hipGetLastError());
	return 0;
}

template <class T, bool GATED, int TM, int TN, int DEPTH = 2>
static int q8_tile(MmArgs A, const MmEpiOut<T, true>& epi, hipStream_t stream) {
	typedef MmShape<int8_t, TM, TN, 2, TM == 256 ? 4 : 2, DEPTH, GATED, true> Shape;
	A.tilesM = (int32_t) ((A.M + TM - 1) / TM);
	A.tilesN = (A.N + (GATED ? TN / 2 : TN) - 1) / (GATED ? TN / 2 : TN);
	auto kernel = k_mm<Shape, MmEpiOut<T, true>>;
	CLA_HIP(allow_full_lds((const void*) kernel));
	kernel<<<(unsigned) ((int64_t) A.tilesM * A.tilesN), Shape::THREADS, Shape::template lds<MmEpiOut<T, true>>(), stream>>>(A, epi);
	CLA_HIP(hipGetLastError());
	return 0;
}

template <class T, bool GATED>
static int q8_mm(const Q8Product& p, hipStream_t stream) {
	const int N = GATED ? p.N / 2 : p.N; // columns of the output
	if(mm_few_suits<int8_t>(p.m, N, g_numCU))
		return q8_few<T, GATED>(Q8Few<T>{p.W, p.ldW, p.t, p.Q, p.ldQ, p.s, (int32_t) p.m, p.K, N, p.act, (const T*) p.bias, (T*) p.out, p.ldOut, (const T*) p.Y, p.ldY}, stream);
	MmArgs A{};
	A.rows = (const char*) p.Q; A.ldRows = p.ldQ;
	A.cols = (const char*) p.W; A.ldCols = p.ldW;
	A.M = p.m; A.N = N; A.K = A.kPart = (p.K + 15) / 16 * 16; A.parts = 1;
	const MmEpiOut<T, true> epi{p.s, p.t, (const T*) p.bias, (T*) p.out, p.ldOut, p.act,
		(((uintptr_t) p.out | (uintptr_t) (p.ldOut * sizeof(T))) & 15) == 0, 0};
	const int64_t n = GATED ? 2 * (int64_t) N : N, big = ((p.m + 255) / 256) * ((n + 255) / 256), mid = ((p.m + 127) / 128) * ((n + 127) / 128);
	if(big >= g_numCU) return q8_tile<T, GATED, 256, 256>(A, epi, stream);
	if(mid >= g_numCU) return q8_tile<T, GATED, 128, 128>(A, epi, stream);
	if(((p.m + 63) / 64) * ((n + 127) / 128) <= g_numCU) return q8_tile<T, GATED, 64, 128, 4>(A, epi, stream); // (a CU for itself: four steps in LDS)
	return q8_tile<T, GATED, 64, 128>(A, epi, stream);
}

bool q8_fuses(int64_t m, int64_t K) { return m <= Q8_FUSE && m * ((K + 15) & ~(int64_t) 15) <= Q8_FUSE_LDS; }

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
