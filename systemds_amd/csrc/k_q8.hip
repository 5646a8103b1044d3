// 8-bit products with a scale for each row of Y and each column of W:
//   out[i, j] = (sum_k q[i, k] * w[k, j]) * s[i] * t[j] (+ bias[j]),   q[i, k] = Y[i, k] / s[i] to the nearest whole number, s[i] = max |Y[i, :]| * (1 / 127)
// and the gated unit act(out of the first half of the columns) * (out of the second half), one kernel. The sums of 8-bit products are exact in 32 bits
// (at most 131,071 terms of 128 * 128), so an output carries the roundings of its scales' products and its own.
//
// Bound, and what was measured (bf16 rows unless said otherwise). Few rows: the bytes of the weights, 1 x 4096 into 2 x 12288 26 us (3.9 TB/s; 30 us with weights that no cache holds), 1 x 4096 into 4096 6.3 us (the launch and two
// round trips to memory). Many: tiles of 256 x 256, 4096 x 4096 into 2 x 12288 gated 381 - 399 us with 13 of them for the rows' quantisation (2.1 POP/s; the matrix cores are
// busy 55 % of the cycles at 1.85 GHz), 8192 x 8192 into 8192 511 - 530 us. A short sum and a wide result: the result's bytes, 100,003 x 100 into 512 fp64 84 us (4.9 TB/s) behind 31 us of quantisation.
#include "../../include/cla_hip.h"
#include "k_q8.hpp"
#include "k_mm_out.hpp"
#include <algorithm>
#include <cmath>

namespace cla {

// ---- rows to 8 bits ----

// Largest magnitude so far, with whatever is not finite above all that is. fp32: the bits without the sign, as a whole number.
__device__ __forceinline__ uint32_t q8_more(float x, uint32_t m) { return max(m, __float_as_uint(x) & 0x7fffffffu); }
__device__ __forceinline__ double q8_more(double x, double m) {
	const double a = fabs(x);
	return a <= 1.7976931348623157e308 ? fmax(a, m) : (double) INFINITY;
}
__device__ __forceinline__ float q8_value(uint32_t m) { return __uint_as_float(m); }
__device__ __forceinline__ float q8_value(double m) { return (float) m; }

// The scale of a row: the largest times 1 / 127, both in fp32. A row with a value that is not finite, or whose largest is none in fp32, has the scale NaN (and
// zeros): its outputs are NaN.
template <class M>
__device__ __forceinline__ float q8_scale(M largest) {
	const float a = q8_value(largest);
	return a <= 3.4028234663852886e38f ? a * (1.0f / 127.0f) : NAN;
}

// What turns a row's values into whole numbers.
template <class C> struct Q8Row {
	C s, inv, half;
	bool none, wide; // a row of zeros or one with the scale NaN; a scale whose reciprocal or last place leaves fp32's range
	__device__ __forceinline__ explicit Q8Row(float scale) : s((C) scale), inv(C(1) / (C) scale), half(C(0.5) * (C) scale), none(!(scale > 0.0f)), wide(scale < 1e-30f) {}
};

// 16 bytes of a row (V values), `left` values of them there (the others 0)
template <class T> struct Q8Piece {
	static constexpr int V = 16 / (int) sizeof(T);
	typedef typename MmCalc<T>::type C;
	typedef typename std::conditional<std::is_same<C, double>::value, double, uint32_t>::type M;
	struct Vals { T x[V]; };
	static __device__ __forceinline__ mm_i32x4 load(const T* p, int64_t left) { return mm_load16<sizeof(T)>((const char*) p, left * (int) sizeof(T)); }
	static __device__ __forceinline__ C value(const mm_i32x4& p, int v) { return (C) __builtin_bit_cast(Vals, p).x[v]; }
	static __device__ __forceinline__ M largest(const mm_i32x4& p, M m) {
#pragma unroll
		for(int v = 0; v < V; v++) m = q8_more(value(p, v), m);
		return m;
	}
	// x / s to the nearest whole number r, ties to even, as the exact quotient rounds. Adding 1.5 * 2^23 (2^52) to x * (1 / s) leaves a number within one of it in
	// the last bits. x - r s is exact next to s / 2 (both are multiples of x's or half of s's last place, below 2^24 or 2^53 of those): where it is below s / 2 in all
	// of the piece, which is all but always, that is r. Otherwise the comparison decides value by value, and for scales out of range the quotient in fp64, whose
	// distance from a half no fp32 operands can lose.
	static __device__ __forceinline__ MmPack<int8_t, V> whole(const mm_i32x4& p, const Q8Row<C>& row) {
		constexpr C BIG = std::is_same<C, double>::value ? C(6755399441055744.0) : C(12582912.0f);
		MmPack<int8_t, V> o;
		C far = C(0);
#pragma unroll
		for(int v = 0; v < V; v++) {
			const C x = value(p, v), t = fma(x, row.inv, BIG), d = fma(BIG - t, row.s, x);
			far = fmax(far, fabs(d));
			o.x[v] = (int8_t) low(t);
		}
		if(far < row.half && !row.wide) return o;
#pragma unroll
		for(int v = 0; v < V; v++) {
			const C x = value(p, v);
			if(row.none) o.x[v] = 0;
			else if(row.wide) o.x[v] = (int8_t) (int) fmin(fmax(rint((double) x / (double) row.s), -127.0), 127.0);
			else {
				C r = rint(x * row.inv);
				const C d = fma(-r, row.s, x);
				const bool odd = ((int) r & 1) != 0;
				if(d > row.half || (d == row.half && odd)) r += C(1);
				else if(d < -row.half || (d == -row.half && odd)) r -= C(1);
				o.x[v] = (int8_t) (int) fmin(fmax(r, C(-127)), C(127));
			}
		}
		return o;
	}
	static __device__ __forceinline__ uint32_t low(float t) { return __float_as_uint(t); }
	static __device__ __forceinline__ uint32_t low(double t) { return (uint32_t) (unsigned long long) __double_as_longlong(t); }
};

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
	typename P::M largest = 0;
#pragma unroll
	for(int i = 0; i < NV; i++) largest = P::largest(x[i], largest);
	for(int k = (NV * TPR + t) * V; k < K; k += TPR * V) largest = P::largest(P::load(y + k, K - k), largest);
#pragma unroll
	for(int d = (TPR < 64 ? TPR : 64) / 2; d > 0; d >>= 1) {
		const auto o = __shfl_xor(largest, d, 64);
		largest = o > largest ? o : largest;
	}
	if(TPR > 64) {
		__shared__ typename P::M part[4];
		if((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = largest;
		__syncthreads();
#pragma unroll
		for(int i = 0; i < 4; i++) largest = part[i] > largest ? part[i] : largest;
	}
	if(row >= m) return;
	const float s = q8_scale(largest);
	if(t == 0) scale[row] = s;
	int8_t* const q = Q + row * ldQ;
	const Q8Row<C> how(s);
	auto put = [&](int k, const mm_i32x4& p) {
		const MmPack<int8_t, V> o = P::whole(p, how);
		if(k + V <= K) mm_put(q + k, o);
		else {
#pragma unroll
			for(int v = 0; v < V; v++)
				if(k + v < K) q[k + v] = o.x[v];
		}
	};
#pragma unroll
	for(int i = 0; i < NV; i++)
		if(i == 0 || i * TPR * V < K) put((i * TPR + t) * V, x[i]);
	for(int k = (NV * TPR + t) * V; k < K; k += TPR * V) put(k, P::load(y + k, K - k));
}

template <class T>
static int q8_rows(const void* Yp, int64_t m, int K, int64_t ld, int8_t* Q, int64_t ldQ, float* scale, hipStream_t stream) {
	if(m == 0) return 0;
	constexpr int V = 16 / (int) sizeof(T);
	const T* const Y = (const T*) Yp;
	// Short rows 16 threads each, 16 rows a block; up to 2 pieces a lane a wave holds the row and no barrier is needed; longer ones take a block, few rows, too
	// (idle waves would be all they leave).
	const int64_t pieces = (K + V - 1) / V;
#define Q8_ROWS(TPR, NV) \
	for(int64_t r = 0, rows = LAUNCH_THREADS / 256 * (256 / TPR); r < m; r += rows) \
		k_q8_rows<T, TPR, NV><<<(unsigned) ((std::min(m - r, rows) + 256 / TPR - 1) / (256 / TPR)), 256, 0, stream>>>(Y + r * ld, std::min(m - r, rows), K, ld, Q + r * ldQ, ldQ, scale + r)
	if(pieces <= 16) { Q8_ROWS(16, 1); }
	else if(pieces <= 64) { Q8_ROWS(16, 4); }
	else if(m < 1024 || pieces > 64 * 2) {
		if(pieces <= 256 * 2) { Q8_ROWS(256, 2); }
		else if(pieces <= 256 * 4) { Q8_ROWS(256, 4); }
		else { Q8_ROWS(256, 8); }
	}
	else { Q8_ROWS(64, 2); }
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

// The source has a row per column already: 16 bytes a thread (4096 x 4096 147 us value by value, 12 so).
__global__ __launch_bounds__(256) void k_q8_pad(const int8_t* __restrict__ src, int64_t ld, int64_t K, int64_t N, int8_t* __restrict__ W, int64_t ldW) {
	const int64_t per = ldW / 16, n = N * per;
	for(int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t) gridDim.x * 256) {
		const int64_t col = i / per, k = i % per * 16;
		*(mm_i32x4*) (W + col * ldW + k) = mm_load16<1>((const char*) src + col * ld + k, K - k);
	}
}

// The source is row-major: 64 x 64 values through LDS.
__global__ __launch_bounds__(256) void k_q8_layout(const int8_t* __restrict__ src, int64_t ld, int64_t K, int N, int8_t* __restrict__ W, int64_t ldW) {
	__shared__ int8_t tile[64][65];
	const int64_t k0 = (int64_t) blockIdx.x * 64;
	const int n0 = blockIdx.y * 64;
	for(int i = threadIdx.x; i < 4096; i += 256) {
		const int a = i >> 6, b = i & 63;
		tile[b][a] = n0 + b < N && k0 + a < K ? src[(k0 + a) * ld + n0 + b] : (int8_t) 0;
	}
	__syncthreads();
	for(int i = threadIdx.x; i < 4096; i += 256) {
		const int a = i >> 6, b = i & 63;
		if(n0 + a < N) W[(int64_t) (n0 + a) * ldW + k0 + b] = tile[a][b]; // (ldW is a multiple of 128)
	}
}

int launch_q8_layout(const int8_t* src, int64_t ld, int byColumn, int64_t K, int N, int8_t* W, int64_t ldW, hipStream_t stream) {
	if(byColumn) k_q8_pad<<<(unsigned) std::min<int64_t>((ldW / 16 * N + 255) / 256, (int64_t) g_numCU * 16), 256, 0, stream>>>(src, ld, K, N, W, ldW);
	else k_q8_layout<<<dim3((unsigned) (ldW / 64), (unsigned) ((N + 63) / 64)), 256, 0, stream>>>(src, ld, K, N, W, ldW);
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
			__shared__ typename P::M part[Q8_FUSE][MMF_WAVES];
			mm_i32x4 x[Q8_FUSE][NV];
#pragma unroll
			for(int r = 0; r < Q8_FUSE; r++) {
				if(r >= A.m) break; // (uniform)
#pragma unroll
				for(int i = 0; i < NV; i++) x[r][i] = P::load(A.Y + r * A.ldY + (i * NT + tid) * V, A.K - (i * NT + tid) * V);
			}
#pragma unroll
			for(int r = 0; r < Q8_FUSE; r++) {
				if(r >= A.m) break;
				typename P::M big = 0;
#pragma unroll
				for(int i = 0; i < NV; i++) big = P::largest(x[r][i], big);
				for(int k = (NV * NT + tid) * V; k < A.K; k += NT * V) big = P::largest(P::load(A.Y + r * A.ldY + k, A.K - k), big);
#pragma unroll
				for(int d = 32; d > 0; d >>= 1) {
					const auto o = __shfl_xor(big, d, 64);
					big = o > big ? o : big;
				}
				if(lane == 0) part[r][wave] = big;
			}
			__syncthreads();
#pragma unroll
			for(int r = 0; r < Q8_FUSE; r++) {
				if(r >= A.m) break;
				typename P::M most = part[r][0];
#pragma unroll
				for(int w = 1; w < MMF_WAVES; w++) most = part[r][w] > most ? part[r][w] : most;
				const float s = q8_scale(most);
				if(tid == 0) scales[r] = s;
				const Q8Row<C> how(s);
				// (what lies behind the row is 0: so are the piece's bytes)
				auto put = [&](int k, const mm_i32x4& p) { *(MmPack<int8_t, V>*) (q8_smem + SUMS + r * pitch + k) = P::whole(p, how); };
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
			x[h] = mm_scaled<C>((C) sum, (C) s, (C) A.t[col + h * A.N]);
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
	else if(MR == 3) k_q8_few<T, GATED, 3, false><<<grid, 64 * MMF_WAVES, lds, stream>>>(A);
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
	const MmEpiOut<T, true> epi{p.s, p.t, (const T*) p.bias, (T*) p.out, p.ldOut, p.act, 0};
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
