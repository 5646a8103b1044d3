// Gated units act(Y t(Wg) + bg) * (Y t(Wu) + bu) of one type T and their gradients.
//
// Forward: one kernel; a tile holds as many columns of either projection, a wave both values of an output, so the activation and the product are its
// epilogue. 16-bit operands are summed in fp32, fp32 in fp32, fp64 in fp64.
// Backward: the projections again (cheaper than 2 nRowY x nOut values kept by every layer between the passes), with dG and dU as the epilogue, then
//   dY = [dG dU] [Wg; Wu],   dW = t([dG dU]) Y,   db = column sums of [dG dU].
// The tiles want both operands by rows of the summed index, so dG and dU are written by row and by column, W and Y are transposed into the workspace. dG and dU are
// rounded to T between the products: the matrix cores take no wider operand, and a rounding of 2^-9 (bf16) of each of many terms leaves less than the result's own.
// Sums over the batch for few weights are split into parts, joined in their order: results do not depend on timing.
#pragma once
#include "../../include/cla_hip.h"
#include "k_gate.hpp"
#include "k_mm_out.hpp"
#include <algorithm>

namespace cla {

template <class T> struct GateFew {
	const T* Y;
	int64_t ldY;
	const T* W;
	int64_t ldW;
	int32_t m, nIn, nOut, act;
	const T* bias;
	T* out;
	int64_t ld;
};

// Few rows: a stream of the weights (k_mm.hpp); the sums of the block's waves meet in LDS.
template <class T, int MR>
__global__ __launch_bounds__(64 * MMF_WAVES) void k_gate_few(GateFew<T> A) {
	extern __shared__ __attribute__((aligned(16))) char gate_smem[]; // [wave][half][row][column]
	typedef typename MmCalc<T>::type C;
	typedef typename MmOp<T>::Acc16 Acc;
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n0 = blockIdx.x * 16;
	Acc acc[2][MR];
	auto rowOf = [&](int row, int64_t k, int64_t left) { return mm_load16<sizeof(T)>((const char*) (A.Y + (row < A.m ? row : 0) * A.ldY) + k, row < A.m ? left : 0); };
	mm_few<T, true, MR>((const char*) A.W, A.ldW * (int64_t) sizeof(T), n0, A.nOut, (int64_t) A.nIn * sizeof(T), rowOf, [] {}, acc, wave, lane);
	C* const red = (C*) gate_smem;
#pragma unroll
	for(int h = 0; h < 2; h++)
#pragma unroll
		for(int j = 0; j < MR; j++)
#pragma unroll
			for(int r = 0; r < 4; r++) red[((wave * 2 + h) * MR * 16 + 16 * j + (lane & 15)) * 16 + mm_col16<T>(lane, r)] = acc[h][j][r];
	__syncthreads();
	for(int i = threadIdx.x; i < A.m * 16; i += 64 * MMF_WAVES) {
		const int row = i >> 4, col = n0 + (i & 15);
		if(col >= A.nOut) continue;
		C x[2];
#pragma unroll
		for(int h = 0; h < 2; h++) {
			x[h] = C(0);
#pragma unroll
			for(int w = 0; w < MMF_WAVES; w++) x[h] += red[(w * 2 + h) * MR * 256 + i];
			if(A.bias) x[h] += (C) A.bias[col + h * A.nOut];
		}
		A.out[row * A.ld + col] = (T) (mm_act<T>(x[0], A.act) * x[1]);
	}
}

template <class T>
static int gate_few(const GateFew<T>& A, hipStream_t stream) {
	const unsigned grid = (unsigned) ((A.nOut + 15) / 16);
	const int MR = A.m <= 16 ? 1 : A.m <= 32 ? 2 : 4;
	const size_t lds = (size_t) MMF_WAVES * 2 * MR * 256 * sizeof(typename MmCalc<T>::type);
	auto kernel = MR == 1 ? k_gate_few<T, 1> : MR == 2 ? k_gate_few<T, 2> : k_gate_few<T, 4>;
	if(lds > 65536) CLA_HIP(allow_full_lds((const void*) kernel));
	kernel<<<grid, 64 * MMF_WAVES, lds, stream>>>(A);
	CLA_HIP(hipGetLastError());
	return 0;
}

template <class T, int TM, int TN, bool GATED, bool DIRECT, class Epi>
static int gate_tile(MmArgs A, const Epi& epi, hipStream_t stream) {
	constexpr int WM = 2, WN = TM == 256 ? 4 : 2, NF = TN / WN / MmOp<T>::FR;
	constexpr size_t lds = std::max(2 * (TM + TN) * 128, WM * WN * Epi::template region<T, NF, GATED>());
	A.tilesM = (int32_t) ((A.M + TM - 1) / TM);
	A.tilesN = (A.N + (GATED ? TN / 2 : TN) - 1) / (GATED ? TN / 2 : TN);
	const int64_t grid = (int64_t) A.tilesM * A.tilesN * A.parts;
	if(grid > 0x7fffffffLL) { set_error("gate: a product of %lld tiles", (long long) grid); return -CLA_ERR_UNSUPPORTED; }
	auto kernel = k_mm<T, TM, TN, WM, WN, GATED, DIRECT, Epi>;
	CLA_HIP(allow_full_lds((const void*) kernel));
	kernel<<<(unsigned) grid, 64 * WM * WN, lds, stream>>>(A, epi);
	CLA_HIP(hipGetLastError());
	return 0;
}

// Operands whose rows go to LDS without registers
static inline bool gate_direct(const MmArgs& A) {
	return (((uintptr_t) A.rows | (uintptr_t) A.cols | (uintptr_t) A.ldRows | (uintptr_t) A.ldCols | (uintptr_t) A.K) & 15) == 0 && A.ldRows <= MM_MAX_LD &&
		A.ldCols <= MM_MAX_LD;
}

// Rows of a tile: the largest tile of which there are enough for the chip.
template <class T>
static int gate_tile_rows(const MmArgs& A, bool gated) {
	const int64_t n = gated ? 2 * (int64_t) A.N : A.N;
	auto tiles = [&](int tm, int tn) { return ((A.M + tm - 1) / tm) * ((n + tn - 1) / tn) * A.parts; };
	if(sizeof(T) == 2 && gate_direct(A) && tiles(256, 256) >= g_numCU) return 256;
	return tiles(128, 128) >= g_numCU ? 128 : 64;
}

template <class T, bool GATED, class Epi>
static int gate_mm(const MmArgs& A, const Epi& epi, hipStream_t stream) {
	const int rows = gate_tile_rows<T>(A, GATED);
	if(gate_direct(A)) {
		if constexpr(sizeof(T) == 2) {
			if(rows == 256) return gate_tile<T, 256, 256, GATED, true>(A, epi, stream);
		}
		return rows == 128 ? gate_tile<T, 128, 128, GATED, true>(A, epi, stream) : gate_tile<T, 64, 128, GATED, true>(A, epi, stream);
	}
	if constexpr(GATED) // (the other products read what this file has laid out)
		return rows == 128 ? gate_tile<T, 128, 128, GATED, false>(A, epi, stream) : gate_tile<T, 64, 128, GATED, false>(A, epi, stream);
	set_error("gate: operands of a product in the workspace are not aligned");
	return -CLA_ERR_STATE;
}

template <class T>
static MmArgs gate_args(const GateCall& c) {
	MmArgs A{};
	A.rows = (const char*) c.Y; A.ldRows = c.ldY * (int64_t) sizeof(T);
	A.cols = (const char*) c.W; A.ldCols = c.ldW * (int64_t) sizeof(T);
	A.M = c.m; A.N = c.nOut; A.K = A.kPart = (int64_t) c.nIn * sizeof(T); A.parts = 1;
	return A;
}

template <class T>
static bool whole(const void* p, int64_t ld) { return (((uintptr_t) p | (uintptr_t) (ld * (int64_t) sizeof(T))) & 15) == 0; }

constexpr int GATE_FEW = 64;

template <class T>
int gate_forward(const GateCall& c, hipStream_t stream) {
	if(c.m <= GATE_FEW)
		return gate_few<T>(GateFew<T>{(const T*) c.Y, c.ldY, (const T*) c.W, c.ldW, (int32_t) c.m, c.nIn, c.nOut, c.act, (const T*) c.bias, (T*) c.out, c.ldOut}, stream);
	const MmEpiOut<T, false> epi{nullptr, nullptr, (const T*) c.bias, (T*) c.out, c.ldOut, c.act, whole<T>(c.out, c.ldOut), 0};
	return gate_mm<T, true>(gate_args<T>(c), epi, stream);
}

// dst[part][c][r] = src[part * kPart + r][c] for rows r < R, zeros behind them up to padR. Bound: the bytes once in, once out.
template <class U>
__global__ __launch_bounds__(256) void k_mm_transpose(const U* __restrict__ src, int64_t ld, int64_t R, int Cn, U* __restrict__ dst, int64_t ldDst, int64_t zDst,
	int64_t padR, int64_t kPart) {
	__shared__ U tile[64][64 + 4 / sizeof(U) + 1];
	const int64_t r0 = (int64_t) blockIdx.x * 64;
	const int c0 = blockIdx.y * 64;
	const int a = threadIdx.x & 63, b = threadIdx.x >> 6;
	for(int i = b; i < 64; i += 4) tile[i][a] = r0 + i < R && c0 + a < Cn ? src[(r0 + i) * ld + c0 + a] : (U) 0;
	__syncthreads();
	const int64_t part = r0 / kPart, at = r0 - part * kPart;
	if(r0 + a < padR)
		for(int i = b; i < 64; i += 4)
			if(c0 + i < Cn) dst[part * zDst + (int64_t) (c0 + i) * ldDst + at + a] = tile[a][i];
}

// out = the sum of the parts, in their order
template <class T>
__global__ __launch_bounds__(256) void k_mm_join(const typename MmCalc<T>::type* __restrict__ part, int parts, int64_t rows, int cols, T* __restrict__ out, int64_t ld) {
	typedef typename MmCalc<T>::type C;
	const int64_t n = rows * cols;
	for(int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t) gridDim.x * 256) {
		C s = C(0);
		for(int p = 0; p < parts; p++) s += part[p * n + i];
		out[i / cols * ld + i % cols] = (T) s;
	}
}

// Column sums of rows of partial sums: 64 columns a block, its 16 waves every 16th row, joined in the order of the waves.
template <class T>
__global__ __launch_bounds__(1024) void k_gate_sums(const typename MmCalc<T>::type* __restrict__ part, int rows, int cols, T* __restrict__ out) {
	typedef typename MmCalc<T>::type C;
	__shared__ C red[16][64];
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.x * 64 + lane;
	C s = C(0);
	if(col < cols)
		for(int r = wave; r < rows; r += 16) s += part[(int64_t) r * cols + col];
	red[wave][lane] = s;
	__syncthreads();
	if(wave == 0 && col < cols) {
#pragma unroll
		for(int w = 1; w < 16; w++) s += red[w][lane];
		out[col] = (T) s;
	}
}

template <class T>
__global__ __launch_bounds__(256) void k_gate_zero(T* __restrict__ p, int64_t rows, int cols, int64_t ld) {
	for(int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x; i < rows * cols; i += (int64_t) gridDim.x * 256) p[i / cols * ld + i % cols] = (T) 0.0f;
}

template <class T> struct MmBits;
template <> struct MmBits<double> { typedef uint64_t type; };
template <> struct MmBits<float> { typedef uint32_t type; };
template <> struct MmBits<__bf16> { typedef uint16_t type; };
template <> struct MmBits<_Float16> { typedef uint16_t type; };

template <class T>
static int gate_transpose(const void* src, int64_t ld, int64_t R, int Cn, void* dst, int64_t ldDst, int64_t zDst, int64_t padR, int64_t kPart, hipStream_t stream) {
	typedef typename MmBits<T>::type U;
	k_mm_transpose<U><<<dim3((unsigned) ((padR + 63) / 64), (unsigned) ((Cn + 63) / 64)), 256, 0, stream>>>((const U*) src, ld, R, Cn, (U*) dst, ldDst, zDst, padR, kPart);
	CLA_HIP(hipGetLastError());
	return 0;
}

template <class T>
int gate_backward(const GateCall& c, hipStream_t stream) {
	typedef typename MmCalc<T>::type C;
	constexpr int64_t es = sizeof(T), V = 16 / es;
	const int64_t F = c.nOut;
	int rc;
	if(c.m == 0) {
		if(c.dW) k_gate_zero<T><<<(unsigned) std::min<int64_t>((2 * F * c.nIn + 255) / 256, g_numCU * 8), 256, 0, stream>>>((T*) c.dW, 2 * F, c.nIn, c.ldDW);
		if(c.dB) k_gate_zero<T><<<(unsigned) ((2 * F + 255) / 256), 256, 0, stream>>>((T*) c.dB, 1, (int) (2 * F), 2 * F);
		CLA_HIP(hipGetLastError());
		return 0;
	}
	const GatePlan p = gate_plan(c.type, c.m, c.nIn, c.nOut);
	T* const P = (T*) (c.ws + p.P);
	T* const Pt = (T*) (c.ws + p.Pt);
	T* const Wt = (T*) (c.ws + p.Wt);
	T* const Yt = (T*) (c.ws + p.Yt);
	C* const sums = (C*) (c.ws + p.sums);
	const MmEpiBack<T> back{(const T*) c.bias, (const T*) c.D, c.ldD, c.dY ? P : nullptr, 2 * p.half, c.dW ? Pt : nullptr, p.kPart, c.dB ? sums : nullptr, c.act,
		whole<T>(c.D, c.ldD)};
	const MmArgs again = gate_args<T>(c);
	if((rc = gate_mm<T, true>(again, back, stream))) return rc;
	if(c.dB) {
		const int waveRows = gate_tile_rows<T>(again, true) / 2, rows = (int) ((c.m + waveRows - 1) / waveRows); // (a row of partial sums per wave)
		k_gate_sums<T><<<(unsigned) ((2 * F + 63) / 64), 1024, 0, stream>>>(sums, rows, (int) (2 * F), (T*) c.dB);
		CLA_HIP(hipGetLastError());
	}
	if(c.dY) {
		for(int h = 0; h < 2; h++)
			if((rc = gate_transpose<T>((const T*) c.W + h * F * c.ldW, c.ldW, F, c.nIn, Wt + h * p.half, 2 * p.half, 0, p.half, (int64_t) 1 << 40, stream))) return rc;
		MmArgs A{};
		A.rows = (const char*) P; A.ldRows = 2 * p.half * es;
		A.cols = (const char*) Wt; A.ldCols = 2 * p.half * es;
		A.M = c.m; A.N = c.nIn; A.K = A.kPart = 2 * p.half * es; A.parts = 1;
		const MmEpiOut<T, false> epi{nullptr, nullptr, nullptr, (T*) c.dY, c.ldDY, ACT_NONE, whole<T>(c.dY, c.ldDY), 0};
		if((rc = gate_mm<T, false>(A, epi, stream))) return rc;
	}
	if(c.dW) {
		const int64_t pad = (c.m + V - 1) / V * V;
		if((rc = gate_transpose<T>(c.Y, c.ldY, c.m, c.nIn, Yt, p.kPart, c.nIn * p.kPart, pad, p.kPart, stream))) return rc;
		MmArgs A{};
		A.rows = (const char*) Pt; A.ldRows = p.kPart * es; A.zRows = 2 * F * p.kPart * es;
		A.cols = (const char*) Yt; A.ldCols = p.kPart * es; A.zCols = c.nIn * p.kPart * es;
		A.M = 2 * F; A.N = c.nIn; A.K = pad * es; A.kPart = p.kPart * es; A.parts = p.parts;
		if(p.parts == 1) {
			const MmEpiOut<T, false> epi{nullptr, nullptr, nullptr, (T*) c.dW, c.ldDW, ACT_NONE, whole<T>(c.dW, c.ldDW), 0};
			return gate_mm<T, false>(A, epi, stream);
		}
		C* const joins = (C*) (c.ws + p.joins);
		const MmEpiOut<C, false> epi{nullptr, nullptr, nullptr, joins, c.nIn, ACT_NONE, whole<C>(joins, c.nIn), 2 * F * c.nIn};
		if((rc = gate_mm<T, false>(A, epi, stream))) return rc;
		k_mm_join<T><<<(unsigned) std::min<int64_t>((2 * F * c.nIn + 255) / 256, g_numCU * 8), 256, 0, stream>>>(joins, p.parts, 2 * F, c.nIn, (T*) c.dW, c.ldDW);
		CLA_HIP(hipGetLastError());
	}
	return 0;
}

} // namespace cla
