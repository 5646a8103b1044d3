// Gated units act(Y t(Wg) + bg) * (Y t(Wu) + bu) of one type T and their gradients.
//
// Forward: one kernel; a tile holds as many columns of either projection, a wave both values of an output, so the activation and the product are its
// epilogue. 16-bit operands are summed in fp32, fp32 in fp32, fp64 in fp64.
// Backward, three or four launches: the projections again (cheaper than 2 nRowY x nOut values kept by every layer between the passes), with dG and dU as the epilogue; then
//   dY = [dG dU] [Wg; Wu],   dW = t([dG dU]) Y,   db = column sums of [dG dU]
// together; then the sums that were split.
// The tiles want both operands by rows of the summed index, so dG and dU are written by row and by column, W and Y are transposed into the workspace. dG and dU are
// rounded to T between the products: the matrix cores take operands of 16 bits at 8 times the rate of fp32, and both operands of one type. Independent roundings of a sum's terms leave as much, relative to
// the result, as one of the result does, so the gradients of Y and W are off by 1.4 times the latter alone (bf16, 2-norm: 0.0023 of 0.0017); as a sum of two 16-bit values each the two products would take
// twice their time, two thirds of the call. fp16 has too few exponents for that: a row (for dY) or column (for dW) of them is brought into range by a power of two that the product takes back.
// Sums over the batch for few weights are split into parts, joined in their order: results do not depend on timing.
//
// Bound, and what was measured. Few rows: the bytes of the weights, bf16 4 x 4096 into 2 x 12288 39 us (5.2 TB/s). Many: the tiles (k_mm.hpp), bf16 4096 x 4096 into 2 x 12288 660 - 683 us
// (1.25 PFLOP/s), gradients at 2 x 8192 1477 - 1573 us: layouts 65, projections 550, both products 960. fp64 400,009 x 100 into 2 x 64 245 - 250 us: 133 of matrix instructions, which the logistic
// function's vector instructions add to.
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
	int64_t m;
	int32_t nIn, nOut, act;
	const T* bias;
	T* out;
	int64_t ld;
	MmEpiBack<T> back;  // BACK: in place of out
};

// Few results: a stream of the weights (k_mm.hpp); the sums of the block's waves meet in LDS.
template <class T, int MR, bool BACK>
__global__ __launch_bounds__(64 * MMF_WAVES) void k_gate_few(GateFew<T> A) {
	extern __shared__ __attribute__((aligned(16))) char gate_smem[]; // [wave][half][row][column]
	typedef typename MmCalc<T>::type C;
	typedef typename MmOp<T>::Acc16 Acc;
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n0 = blockIdx.x * 16;
	const int64_t m0 = (int64_t) blockIdx.y * 16 * MR;
	const int rows = (int) min(A.m - m0, (int64_t) 16 * MR);
	const T* const Y = A.Y + m0 * A.ldY;
	Acc acc[2][MR];
	auto rowOf = [&](int row, int64_t k, int64_t left) { return mm_load16<sizeof(T)>((const char*) (Y + (row < rows ? row : 0) * A.ldY) + k, row < rows ? left : 0); };
	mm_few<T, true, MR>((const char*) A.W, A.ldW * (int64_t) sizeof(T), n0, A.nOut, (int64_t) A.nIn * sizeof(T), rowOf, [] {}, acc, wave, lane);
	C* const red = (C*) gate_smem;
#pragma unroll
	for(int h = 0; h < 2; h++)
#pragma unroll
		for(int j = 0; j < MR; j++)
#pragma unroll
			for(int r = 0; r < 4; r++) red[((wave * 2 + h) * MR * 16 + 16 * j + (lane & 15)) * 16 + mm_col16<T>(lane, r)] = acc[h][j][r];
	__syncthreads();
	for(int i = threadIdx.x; i < (BACK ? 16 * MR : rows) * 16; i += 64 * MMF_WAVES) {
		const int row = i >> 4, col = n0 + (i & 15), at = min(col, A.nOut - 1);
		const bool in = row < rows && col < A.nOut;
		C x[2];
#pragma unroll
		for(int h = 0; h < 2; h++) {
			x[h] = C(0);
#pragma unroll
			for(int w = 0; w < MMF_WAVES; w++) x[h] += red[(w * 2 + h) * MR * 256 + i];
			if(A.bias) x[h] += (C) A.bias[at + h * A.nOut];
		}
		if constexpr(!BACK) {
			if(in) A.out[(m0 + row) * A.ld + col] = (T) (mm_act<T>(x[0], A.act) * x[1]);
		}
		else {
			// (as MmEpiBack: zeros up to whole 16 bytes both ways)
			const MmEpiBack<T>& B = A.back;
			C value, slope;
			mm_act_both<T>(x[0], A.act, value, slope);
			const C d = in ? (C) B.D[(m0 + row) * B.ldD + col] : C(0);
			const C dG = in ? d * x[1] * slope : C(0), dU = in ? d * value : C(0);
			red[i] = dG; red[MR * 256 + i] = dU; // (of the first wave's sums nothing but this thread's are read at this place)
			const int64_t half = B.ldP / 2, m = m0 + row, pad = 16 / (int) sizeof(T);
			if(B.P && row < rows && col < half) {
				const C by = B.row_power(m);
				B.P[m * B.ldP + col] = (T) (dG * by);
				B.P[m * B.ldP + half + col] = (T) (dU * by);
			}
			if(B.Pt && col < A.nOut && m < (A.m + pad - 1) / pad * pad) {
				const int64_t part = m / B.kPart;
				T* const to = B.Pt + part * 2 * A.nOut * B.kPart + (m - part * B.kPart);
				to[col * B.kPart] = (T) (dG * B.col_power(col));
				to[(col + A.nOut) * B.kPart] = (T) (dU * B.col_power(col + A.nOut));
			}
		}
	}
	if constexpr(BACK) {
		if(!A.back.sums) return; // (uniform)
		__syncthreads();
		const int h = threadIdx.x >> 4, c = threadIdx.x & 15;
		if(h < 2 && n0 + c < A.nOut) {
			C s = C(0);
			for(int r = 0; r < rows; r++) s += red[h * MR * 256 + r * 16 + c];
			A.back.sums[(int64_t) blockIdx.y * 2 * A.nOut + h * A.nOut + n0 + c] = s;
		}
	}
}

// Rows to a block, in sixteens (64 rows of fp64 do not fit the registers).
template <class T>
static int gate_few_rows(int64_t m, int nOut) { return std::min(mm_few_rows(m, nOut, g_numCU), sizeof(T) == 8 ? 2 : 4); }

template <class T, bool BACK>
static int gate_few(const GateFew<T>& A, hipStream_t stream) {
	const int MR = gate_few_rows<T>(A.m, A.nOut);
	const dim3 grid((unsigned) ((A.nOut + 15) / 16), (unsigned) ((A.m + 16 * MR - 1) / (16 * MR)));
	const size_t lds = (size_t) MMF_WAVES * 2 * MR * 256 * sizeof(typename MmCalc<T>::type);
	constexpr bool WIDE = sizeof(T) == 8;
	auto kernel = MR == 1 ? k_gate_few<T, 1, BACK> : MR == 2 ? k_gate_few<T, 2, BACK> : MR == 3 ? k_gate_few<T, WIDE ? 2 : 3, BACK> : k_gate_few<T, WIDE ? 2 : 4, BACK>;
	if(lds > 65536) CLA_HIP(allow_full_lds((const void*) kernel));
	kernel<<<grid, 64 * MMF_WAVES, lds, stream>>>(A);
	CLA_HIP(hipGetLastError());
	return 0;
}

// Operands whose rows go to LDS without registers. (16-bit types with odd sizes pass through registers, 2048 x 2047 into 2048 69 us where 2048 x 2046 takes 54 and 2048 x 2048 39; so did every size
// that is no whole 16 bytes before.)
static inline bool gate_direct(const MmArgs& A) {
	return (((uintptr_t) A.rows | (uintptr_t) A.cols | (uintptr_t) A.ldRows | (uintptr_t) A.ldCols | (uintptr_t) A.K) & 3) == 0 && A.ldRows <= MM_MAX_LD &&
		A.ldCols <= MM_MAX_LD;
}

// A tile's shape (TM * 1000 + TN; 64129: 64 x 128 with four steps in LDS, which takes a CU for itself). 16-bit types: the largest of which there is one for every CU
// (fewer, larger tiles read less through LDS, which is what small ones are bound by). fp32 and fp64 are bound by their matrix instructions at any size: the shape whose tiles leave the busiest CU the least.
template <class T>
static int gate_shape(const MmArgs& A, bool gated) {
	const int64_t n = gated ? 2 * (int64_t) A.N : A.N;
	auto tiles = [&](int tm, int tn) { return ((A.M + tm - 1) / tm) * ((n + tn - 1) / tn) * A.parts; };
	if(sizeof(T) == 2) {
		if(gate_direct(A) && (A.K & 15) == 0 && tiles(256, 256) >= g_numCU) return 256256;
		if(tiles(128, 128) >= g_numCU) return 128128;
		return gate_direct(A) && tiles(64, 128) <= g_numCU ? 64129 : 64128;
	}
	int best = 0;
	int64_t least = 0;
	for(const int shape : {128128, 64128, 64064}) {
		const int tm = shape / 1000, tn = shape % 1000;
		const int64_t cost = (tiles(tm, tn) + g_numCU - 1) / g_numCU * tm * tn;
		if(best == 0 || cost < least) { best = shape; least = cost; }
	}
	return best;
}

template <class Shape>
static int64_t gate_tiles(MmArgs& A) {
	constexpr int cols = Shape::GATED ? Shape::TN / 2 : Shape::TN;
	A.tilesM = (int32_t) ((A.M + Shape::TM - 1) / Shape::TM);
	A.tilesN = (A.N + cols - 1) / cols;
	return (int64_t) A.tilesM * A.tilesN * A.parts;
}

static inline int gate_grid(int64_t blocks, int threads) {
	if(blocks <= LAUNCH_THREADS / threads) return 0;
	set_error("gate: a launch of %lld blocks of %d threads (fewer rows at a time)", (long long) blocks, threads);
	return -CLA_ERR_UNSUPPORTED;
}

// Calls launch(Shape()) with the shape of that number.
template <class T, bool GATED, bool DIRECT, class Launch>
static int gate_with(int shape, const Launch& launch) {
	if constexpr(sizeof(T) == 2) {
		if constexpr(DIRECT) {
			if(shape == 256256) return launch(MmShape<T, 256, 256, 2, 4, 2, GATED, DIRECT>());
			if(shape == 64129) return launch(MmShape<T, 64, 128, 2, 2, 4, GATED, DIRECT>());
		}
	}
	else {
		if(shape == 64064) return launch(MmShape<T, 64, 64, 2, 2, 2, GATED, DIRECT>());
	}
	if(shape == 128128) return launch(MmShape<T, 128, 128, 2, 2, 2, GATED, DIRECT>());
	return launch(MmShape<T, 64, 128, 2, 2, 2, GATED, DIRECT>());
}

// The projections of a gated unit, with more blocks of other work behind them.
template <class T, class Epi, class More>
static int gate_project(MmArgs A, const Epi& epi, int64_t moreBlocks, const More& more, hipStream_t stream) {
	const int shape = gate_shape<T>(A, true);
	auto launch = [&](auto s) {
		typedef decltype(s) Shape;
		const int64_t blocks = gate_tiles<Shape>(A);
		if(const int rc = gate_grid(blocks + moreBlocks, Shape::THREADS)) return rc;
		auto kernel = k_mm_and<Shape, Epi, More>;
		CLA_HIP(allow_full_lds((const void*) kernel));
		kernel<<<(unsigned) (blocks + moreBlocks), Shape::THREADS, std::max(Shape::template lds<Epi>(), More::LDS), stream>>>(A, epi, (unsigned) blocks, more);
		CLA_HIP(hipGetLastError());
		return 0;
	};
	return gate_direct(A) ? gate_with<T, true, true>(shape, launch) : gate_with<T, true, false>(shape, launch);
}

struct GateNothing {
	static constexpr size_t LDS = 0;
	__device__ void run(unsigned, char*) const {}
};

template <class T>
static MmArgs gate_args(const GateCall& c) {
	MmArgs A{};
	A.rows = (const char*) c.Y; A.ldRows = c.ldY * (int64_t) sizeof(T);
	A.cols = (const char*) c.W; A.ldCols = c.ldW * (int64_t) sizeof(T);
	A.M = c.m; A.N = c.nOut; A.K = A.kPart = (int64_t) c.nIn * sizeof(T); A.parts = 1;
	return A;
}

template <class T>
int gate_forward(const GateCall& c, hipStream_t stream) {
	if(mm_few_suits<T>(c.m, c.nOut, g_numCU))
		return gate_few<T, false>(GateFew<T>{(const T*) c.Y, c.ldY, (const T*) c.W, c.ldW, c.m, c.nIn, c.nOut, c.act, (const T*) c.bias, (T*) c.out, c.ldOut, {}}, stream);
	const MmEpiOut<T, false> epi{nullptr, nullptr, (const T*) c.bias, (T*) c.out, c.ldOut, c.act, 0};
	return gate_project<T>(gate_args<T>(c), epi, 0, GateNothing(), stream);
}

// dst[part][c][r] = src[part * kPart + r][c] for rows r < R, zeros behind them up to padR; a block takes 64 x 64 of it.
struct GateTranspose {
	const void* src; int64_t ld, R; int32_t cols;
	void* dst; int64_t ldDst, zDst, padR, kPart;
	unsigned blocksR, blocks;   // 0 blocks: nothing to do
	static GateTranspose of(const void* src, int64_t ld, int64_t R, int cols, void* dst, int64_t ldDst, int64_t zDst, int64_t padR, int64_t kPart) {
		const int64_t r = (padR + 63) / 64;
		return {src, ld, R, cols, dst, ldDst, zDst, padR, kPart, (unsigned) r, (unsigned) std::min<int64_t>(r * ((cols + 63) / 64), 0x7fffffffLL)};
	}
};

// The backward pass's other layouts: both halves of t(W) and t(Y). Bound: the bytes once in, once out, 16 of them a lane.
template <class U> struct GateLayouts {
	GateTranspose t[3];
	static constexpr int PITCH = 64 + (sizeof(U) == 2 ? 2 : 1);
	static constexpr size_t LDS = 64 * PITCH * sizeof(U);
	__device__ __forceinline__ void run(unsigned block, char* smem) const {
		constexpr int V = 16 / (int) sizeof(U), PER = 64 / V;
		U* const tile = (U*) smem;
		const int i = block < t[0].blocks ? 0 : block - t[0].blocks < t[1].blocks ? 1 : 2;
		if(i > 0) block -= t[0].blocks;
		if(i > 1) block -= t[1].blocks;
		const GateTranspose g = t[i];
		const U* const src = (const U*) g.src;
		U* const dst = (U*) g.dst;
		const int64_t r0 = (int64_t) (block % g.blocksR) * 64;
		const int c0 = (int) (block / g.blocksR) * 64, a = threadIdx.x % PER * V, step = blockDim.x / PER;
		for(int b = threadIdx.x / PER; b < 64; b += step) {
			MmPack<U, V> p;
			const bool in = r0 + b < g.R;
			const U* const from = src + (r0 + b) * g.ld + c0 + a;
			if(in && c0 + a + V <= g.cols) p = mm_get<MmPack<U, V>>(from);
			else {
#pragma unroll
				for(int v = 0; v < V; v++) p.x[v] = in && c0 + a + v < g.cols ? from[v] : (U) 0;
			}
#pragma unroll
			for(int v = 0; v < V; v++) tile[b * PITCH + a + v] = p.x[v];
		}
		__syncthreads();
		const int64_t part = r0 / g.kPart, at = r0 - part * g.kPart;
		for(int b = threadIdx.x / PER; b < 64; b += step) { // (padR and the rows' starts are multiples of 16 bytes)
			if(c0 + b >= g.cols || r0 + a >= g.padR) continue;
			MmPack<U, V> p;
#pragma unroll
			for(int v = 0; v < V; v++) p.x[v] = tile[(a + v) * PITCH + b];
			*(MmPack<U, V>*) (dst + part * g.zDst + (int64_t) (c0 + b) * g.ldDst + at + a) = p;
		}
	}
};

template <class U, class More>
__global__ __launch_bounds__(256) void k_gate_layouts(GateLayouts<U> lay, unsigned blocks, More more) {
	__shared__ __attribute__((aligned(16))) char smem[GateLayouts<U>::LDS];
	if(blockIdx.x < blocks) lay.run(blockIdx.x, smem);
	else more.run(blockIdx.x - blocks, smem);
}

// Sums of 64 rows of partial sums at a time: a block takes 64 columns of them, its waves 64 rows each.
template <class C> struct GateSums {
	const C* part; C* out;
	int32_t rows, cols, groups;
	unsigned blocksC;
	static constexpr size_t LDS = 0;
	__device__ __forceinline__ void run(unsigned block, char*) const {
		const int col = (int) (block % blocksC) * 64 + (threadIdx.x & 63), group = (int) (block / blocksC) * (blockDim.x / 64) + (threadIdx.x >> 6);
		if(col >= cols || group >= groups) return;
		const int r0 = group * 64, n = min(64, rows - r0);
		const C* const p = part + (int64_t) r0 * cols + col;
		C s = C(0);
#pragma unroll 8
		for(int r = 0; r < n; r++) s += p[(int64_t) r * cols];
		out[(int64_t) group * cols + col] = s;
	}
};

// out = the sum of the parts: a block takes 64 values, each of its waves a quarter of the parts, in their order.
template <class T> struct GateJoin {
	const typename MmCalc<T>::type* part;
	T* out;
	int64_t rows, ld;
	int32_t cols, parts;
	unsigned blocks;            // 0: nothing to do
	static GateJoin of(const typename MmCalc<T>::type* part, T* out, int64_t rows, int cols, int64_t ld, int parts) {
		return {part, out, rows, ld, cols, parts, (unsigned) std::min<int64_t>((rows * cols + 63) / 64, 1 << 20)};
	}
};

template <class T> struct GateJoins { GateJoin<T> j[3]; };

template <class T>
__global__ __launch_bounds__(256) void k_gate_join(GateJoins<T> all) {
	typedef typename MmCalc<T>::type C;
	__shared__ C red[4][64];
	unsigned block = blockIdx.x;
	const int i = block < all.j[0].blocks ? 0 : block - all.j[0].blocks < all.j[1].blocks ? 1 : 2;
	if(i > 0) block -= all.j[0].blocks;
	if(i > 1) block -= all.j[1].blocks;
	const GateJoin<T> g = all.j[i];
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, per = (g.parts + 3) / 4, p0 = min(wave * per, g.parts), p1 = min(p0 + per, g.parts);
	const int64_t n = g.rows * g.cols;
	for(int64_t v0 = (int64_t) block * 64; v0 < n; v0 += (int64_t) g.blocks * 64) {
		const int64_t v = v0 + lane;
		C s = C(0);
		if(v < n) {
#pragma unroll 4
			for(int p = p0; p < p1; p++) s += g.part[p * n + v];
		}
		red[wave][lane] = s;
		__syncthreads();
		if(wave == 0 && v < n) {
#pragma unroll
			for(int w = 1; w < 4; w++) s += red[w][lane];
			g.out[v / g.cols * g.ld + v % g.cols] = (T) s;
		}
		__syncthreads();
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

// fp16: bounds of dG and dU, whose magnitudes may leave the type's range (above, or below where their sums do not) though the gradients do not:
//   |dG| <= 1.13 |D| (|y| |wu| + |bu|),   |dU| <= |D| max(|y| |wg| + bg, 1)
// of the 2-norms of the rows of Y and W (a derivative of an activation is at most 1.13, a value at most its argument or 1, the logistic function's 1; a gate shut by a bias of -infinity bounds nothing;
// without an activation |bg|); up to sqrt(nIn) above what is there, which costs as much of the 2^39 between
// the bound and the last place left. An output that D leaves out (0) bounds nothing.
// Cost, both kernels and the products' rows: 4096 x 4096 into 2 x 8192 63 us of 1605, 4 x 1245 into 977 9 of 38 (the norms behind the layouts; in a launch of their own 103 and 12).
struct GateNorms {
	const _Float16* Y; int64_t m, ldY;
	const _Float16* W; int64_t rowsW, ldW;
	int32_t K;
	float* normY; float* normW;
	uint32_t* mostRow; uint32_t* mostCol;   // cleared on the way
	unsigned blocks;
	template <int TPR> __device__ __forceinline__ void rows(unsigned block) const { // TPR threads to a row
		constexpr int ROWS = 256 / TPR;
		const int t = threadIdx.x % TPR;
		for(int64_t row = (int64_t) block * ROWS + threadIdx.x / TPR; row < m + rowsW; row += (int64_t) blocks * ROWS) {
			const bool ofY = row < m;
			const _Float16* const x = ofY ? Y + row * ldY : W + (row - m) * ldW;
			float s = 0.0f;
			for(int k = t * 8; k < K; k += TPR * 8) {
				const mm_f16x8 p = __builtin_bit_cast(mm_f16x8, mm_load16<2>((const char*) (x + k), (int64_t) (K - k) * 2));
#pragma unroll
				for(int v = 0; v < 8; v++) s = fmaf((float) p[v], (float) p[v], s);
			}
#pragma unroll
			for(int d = TPR / 2; d > 0; d >>= 1) s += __shfl_xor(s, d, TPR);
			if(t == 0) {
				if(ofY) { normY[row] = sqrtf(s); mostRow[row] = 0; }
				else { normW[row - m] = sqrtf(s); mostCol[row - m] = 0; }
			}
		}
	}
	__device__ __forceinline__ void run(unsigned block, char*) const {
		if(K <= 128) rows<16>(block);
		else rows<64>(block);
	}
	static GateNorms of(const GateCall& c, float* normY, float* normW, uint32_t* mostRow, uint32_t* mostCol) {
		const int64_t n = c.m + 2 * (int64_t) c.nOut, perBlock = c.nIn <= 128 ? 16 : 4;
		return {(const _Float16*) c.Y, c.m, c.ldY, (const _Float16*) c.W, 2 * (int64_t) c.nOut, c.ldW, c.nIn, normY, normW, mostRow, mostCol,
			(unsigned) std::min<int64_t>((n + perBlock - 1) / perBlock, g_numCU * 8)};
	}
};

// A block takes 512 columns of `steps` times 64 rows, its waves 8 rows at a time: a block to a CU, since what costs is that they meet at the columns' maxima (4096 x 8192 38 us, a block for every
// 64 rows 57). Rows and columns behind the last ones are the last ones again, which changes no maximum. (A largest magnitude does not depend on the order: the bits of what is not negative, those
// of NaN above all others.) WIDE: rows of 8 values or more.
template <bool WIDE>
__global__ __launch_bounds__(512) void k_gate_bounds(const _Float16* __restrict__ D, int64_t ldD, int64_t m, int N, const _Float16* __restrict__ bias, const float* __restrict__ normY,
	const float* __restrict__ normW, uint32_t* __restrict__ mostRow, uint32_t* __restrict__ mostCol, int64_t steps, int act) {
	__shared__ uint32_t part[8][16][65];
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, colRuns = (N + 511) / 512;
	const int64_t step0 = (int64_t) (blockIdx.x / (unsigned) colRuns) * steps;
	const int first = (int) (blockIdx.x % (unsigned) colRuns) * 512, c0 = WIDE ? min(first + lane * 8, N - 8) : 0;
	float wg[8], wu[8], bg[8], bu[8];
	uint32_t most[16]; // (gate's columns, the other projection's)
#pragma unroll
	for(int v = 0; v < 8; v++) {
		const int c = min(c0 + v, N - 1);
		wg[v] = act == ACT_SIGMOID ? 0.0f : normW[c]; wu[v] = 1.13f * normW[c + N];
		bg[v] = !bias || act == ACT_SIGMOID ? 0.0f : act == ACT_NONE ? fabsf((float) bias[c]) : (float) bias[c]; bu[v] = bias ? 1.13f * fabsf((float) bias[c + N]) : 0.0f;
		most[v] = most[8 + v] = 0;
	}
	for(int64_t step = step0; step < step0 + steps; step++) {
		const int64_t r0 = step * 64 + wave * 8;
		if(r0 >= m) break; // (uniform)
		mm_f16x8 d[8];
		float ny[8];
		uint32_t row[8];
#pragma unroll
		for(int i = 0; i < 8; i++) {
			const int64_t at = min(r0 + i, m - 1);
			if(WIDE) __builtin_memcpy(&d[i], D + at * ldD + c0, 16);
			else {
#pragma unroll
				for(int v = 0; v < 8; v++) d[i][v] = D[at * ldD + min(v, N - 1)];
			}
			ny[i] = normY[at];
		}
#pragma unroll
		for(int i = 0; i < 8; i++) {
			row[i] = 0;
#pragma unroll
			for(int v = 0; v < 8; v++) {
				const float a = fabsf((float) d[i][v]);
				const uint32_t p = __float_as_uint(a * fmaf(ny[i], wu[v], bu[v])), q = __float_as_uint(a * fmaxf(fmaf(ny[i], wg[v], bg[v]), 1.0f));
				most[v] = max(most[v], p); most[8 + v] = max(most[8 + v], q);
				row[i] = max(row[i], max(p, q));
			}
		}
		// the lanes' largest of 8 rows: each half of the lanes keeps half of the rows, three times over; row[0] is that of row lane / 8 in the end
#pragma unroll
		for(int s = 32, n = 4; n > 0; s >>= 1, n >>= 1) {
			const bool high = (lane & s) != 0;
#pragma unroll
			for(int i = 0; i < n; i++) {
				const uint32_t other = (uint32_t) __shfl_xor((int) (high ? row[i] : row[i + n]), s, 64);
				row[i] = max(high ? row[i + n] : row[i], other);
			}
		}
#pragma unroll
		for(int s = 4; s > 0; s >>= 1) row[0] = max(row[0], (uint32_t) __shfl_xor((int) row[0], s, 64));
		if((lane & 7) == 0 && r0 + (lane >> 3) < m && row[0] != 0) atomicMax(mostRow + r0 + (lane >> 3), row[0]);
	}
#pragma unroll
	for(int v = 0; v < 16; v++) part[wave][v][lane] = most[v];
	__syncthreads();
	const int c = first + (int) threadIdx.x; // neighbouring threads, neighbouring columns: an atomic access is a line for 16 of them
	if(c < N) {
		const int l = threadIdx.x >> 3, v = WIDE ? c - min(first + l * 8, N - 8) : c;
#pragma unroll
		for(int h = 0; h < 2; h++) {
			uint32_t x = 0;
#pragma unroll
			for(int w = 0; w < 8; w++) x = max(x, part[w][h * 8 + v][l]);
			if(x != 0) atomicMax(mostCol + h * N + c, x);
		}
	}
}

// Where a product goes: T, or (parts > 1) partial sums. One type for both, so that one kernel holds either product.
template <class T> struct GateOut {
	static constexpr bool POWERS = MmEpiBack<T>::POWERS;
	MmEpiOut<T, false, POWERS> whole;
	MmEpiOut<typename MmCalc<T>::type, false, POWERS> part;
	int32_t parts;
	template <class E, int NF, bool GATED> static constexpr int region() { return MmRegion<E, NF, GATED>::BYTES; }
	template <class E, int MF, int NF, bool GATED, class Acc>
	__device__ __forceinline__ void run(Acc& acc, char* region, int64_t m0, int n0, int64_t M, int N, int p, int rowPart, int lane) const {
		if(parts == 1) whole.template run<E, MF, NF, GATED>(acc, region, m0, n0, M, N, p, rowPart, lane);
		else part.template run<E, MF, NF, GATED>(acc, region, m0, n0, M, N, p, rowPart, lane);
	}
	static GateOut of(T* out, int64_t ld, typename MmCalc<T>::type* joins, int64_t M, int64_t N, int parts, const uint32_t* most) {
		return {{(const float*) most, nullptr, nullptr, out, ld, ACT_NONE, 0},
			{(const float*) most, nullptr, nullptr, joins, N, ACT_NONE, M * N}, parts};
	}
};

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
	typedef typename MmBits<T>::type U;
	const GatePlan p = gate_plan(c.type, c.m, c.nIn, c.nOut);
	T* const P = (T*) (c.ws + p.P);
	T* const Pt = (T*) (c.ws + p.Pt);
	T* const Wt = (T*) (c.ws + p.Wt);
	T* const Yt = (T*) (c.ws + p.Yt);
	C* const sums = (C*) (c.ws + p.sums);
	C* const sums64 = (C*) (c.ws + p.sums64);
	uint32_t* const mostRow = (uint32_t*) (c.ws + p.mostRow);
	uint32_t* const mostCol = (uint32_t*) (c.ws + p.mostCol);
	const int64_t pad = (c.m + V - 1) / V * V;

	// projections, dG and dU; W and Y the other way round
	const MmArgs project = gate_args<T>(c);
	const MmEpiBack<T> back{(const T*) c.bias, (const T*) c.D, c.ldD, c.dY ? P : nullptr, 2 * p.half, c.dW ? Pt : nullptr, p.kPart, c.dB ? sums : nullptr, c.act, mostRow, mostCol};
	GateLayouts<U> lay{};
	const int64_t one = (int64_t) 1 << 40; // (a single part)
	if(c.dY)
		for(int h = 0; h < 2; h++)
			lay.t[h] = GateTranspose::of((const T*) c.W + h * F * c.ldW, c.ldW, F, c.nIn, Wt + h * p.half, 2 * p.half, 0, p.half, one);
	if(c.dW) lay.t[2] = GateTranspose::of(c.Y, c.ldY, c.m, c.nIn, Yt, p.kPart, c.nIn * p.kPart, pad, p.kPart);
	int64_t lays = (int64_t) lay.t[0].blocks + lay.t[1].blocks + lay.t[2].blocks;
	if((rc = gate_grid(lays + g_numCU * 8, 256))) return rc; // (the norms' blocks are at most so many)
	if constexpr(MmEpiBack<T>::POWERS) { // (the layouts ride along with the norms)
		if(c.dY || c.dW) {
			float* const normY = (float*) (c.ws + p.normY);
			float* const normW = (float*) (c.ws + p.normW);
			const GateNorms norms = GateNorms::of(c, normY, normW, mostRow, mostCol);
			k_gate_layouts<U><<<(unsigned) lays + norms.blocks, 256, 0, stream>>>(lay, (unsigned) lays, norms);
			lays = 0;
			auto bounds = F >= 8 ? k_gate_bounds<true> : k_gate_bounds<false>;
			const int64_t colRuns = (F + 511) / 512, rowSteps = (c.m + 63) / 64, steps = (rowSteps * colRuns + g_numCU - 1) / g_numCU;
			bounds<<<(unsigned) ((rowSteps + steps - 1) / steps * colRuns), 512, 0, stream>>>((const T*) c.D, c.ldD, c.m, c.nOut, (const T*) c.bias, normY, normW, mostRow, mostCol, steps, c.act);
			CLA_HIP(hipGetLastError());
		}
	}
	// few of them behind the projections' tiles, in the same launch; many in one of their own: a tile's LDS leaves a CU to one block (4096 x 4096 into 2 x 8192 on
	// bf16 1.85 ms in all, 1.50 so)
	// (so few results that tiles would take a handful of CUs; more are written by column faster from a tile, and the layouts ride along: 59 x 4055 into 174 in fp64 277 us on
	// tiles, 72 so, 76 x 256 into 2560 44 and 53)
	const bool few = (c.m + 15) / 16 * ((F + 15) / 16) <= g_numCU;
	if(lays > (few ? 0 : 2 * g_numCU)) {
		k_gate_layouts<U><<<(unsigned) lays, 256, 0, stream>>>(lay, (unsigned) lays, GateNothing());
		lays = 0;
	}
	if(few) rc = gate_few<T, true>(GateFew<T>{(const T*) c.Y, c.ldY, (const T*) c.W, c.ldW, c.m, c.nIn, c.nOut, c.act, (const T*) c.bias, nullptr, 0, back}, stream);
	else rc = gate_project<T>(project, back, lays, lay, stream);
	if(rc) return rc;

	// dY = P W and dW = t(P) Y; the first sums of dB
	MmArgs A{}, B{};
	A.rows = (const char*) P; A.cols = (const char*) Wt; A.ldRows = A.ldCols = A.K = 2 * p.half * es;
	A.M = c.dY ? c.m : 0; A.N = c.nIn; A.zRows = A.zCols = A.kPart = p.kPartY; A.parts = p.partsY;
	B.rows = (const char*) Pt; B.cols = (const char*) Yt; B.ldRows = B.ldCols = B.kPart = p.kPart * es; B.K = pad * es;
	B.zRows = 2 * F * p.kPart * es; B.zCols = c.nIn * p.kPart * es;
	B.M = c.dW ? 2 * F : 0; B.N = c.nIn; B.parts = p.parts;
	C* const joinsY = (C*) (c.ws + p.joinsY);
	C* const joinsW = (C*) (c.ws + p.joins);
	const GateOut<T> outY = GateOut<T>::of((T*) c.dY, c.ldDY, joinsY, c.m, c.nIn, p.partsY, mostRow), outW = GateOut<T>::of((T*) c.dW, c.ldDW, joinsW, 2 * F, c.nIn, p.parts, mostCol);
	const int waveRows = few ? 16 * gate_few_rows<T>(c.m, c.nOut) : gate_shape<T>(project, true) / 1000 / 2, sumRows = (int) ((c.m + waveRows - 1) / waveRows); // (of a row of partial sums: a block's or a wave's)
	GateSums<C> first{sums, sums64, sumRows, (int32_t) (2 * F), (sumRows + 63) / 64, (unsigned) ((2 * F + 63) / 64)};
	MmArgs both = A; // (the shape that suits both: as many tiles as they have together)
	both.M = A.M * A.parts + B.M * B.parts; both.parts = 1;
	auto launch = [&](auto s) {
		typedef decltype(s) Shape;
		constexpr int waves = Shape::THREADS / 64;
		const int64_t nA = gate_tiles<Shape>(A), nB = gate_tiles<Shape>(B), nC = c.dB ? (int64_t) first.blocksC * ((first.groups + waves - 1) / waves) : 0;
		if(nA + nB + nC == 0) return 0;
		if(const int r = gate_grid(nA + nB + nC, Shape::THREADS)) return r;
		auto kernel = k_mm_two<Shape, GateOut<T>, GateOut<T>, GateSums<C>>;
		CLA_HIP(allow_full_lds((const void*) kernel));
		kernel<<<(unsigned) (nA + nB + nC), Shape::THREADS, Shape::template lds<GateOut<T>>(), stream>>>(A, outY, (unsigned) nA, B, outW, (unsigned) nB, first);
		CLA_HIP(hipGetLastError());
		return 0;
	};
	if((rc = gate_with<T, false, true>(gate_shape<T>(both, false), launch))) return rc;

	GateJoins<T> joins{};
	if(c.dY && p.partsY > 1) joins.j[0] = GateJoin<T>::of(joinsY, (T*) c.dY, c.m, c.nIn, c.ldDY, p.partsY);
	if(c.dW && p.parts > 1) joins.j[1] = GateJoin<T>::of(joinsW, (T*) c.dW, 2 * F, c.nIn, c.ldDW, p.parts);
	if(c.dB) joins.j[2] = GateJoin<T>::of(sums64, (T*) c.dB, 1, (int) (2 * F), 2 * F, first.groups);
	const unsigned blocks = joins.j[0].blocks + joins.j[1].blocks + joins.j[2].blocks;
	if(blocks > 0) k_gate_join<T><<<blocks, 256, 0, stream>>>(joins);
	CLA_HIP(hipGetLastError());
	return 0;
}

} // namespace cla
