// Tiles of a product of two matrices held by rows of the summed index: D[i, j] = sum_k A[i, k] * B[j, k], for 8-bit integers, 16-bit floats,
// fp32 and fp64 alike. "Rows" (i, tokens or table rows) are the output's rows, "columns" (j) its columns: weights, one row of them per column.
//
// All types share one shape of tile, counted in bytes: a step takes 128 bytes of the summed index of every row and column of the tile through
// LDS (128 int8, 64 16-bit, 32 fp32, 16 fp64 values), a lane's matrix operand is 16 bytes of one row. Which values of the summed index meet in
// an instruction does not matter as long as both operands agree, so the fp32 and fp64 instructions, which take one value a lane, run once per
// value of the 16 bytes. Columns are the instruction's A operand, rows its B operand: a lane's results are several columns of one row.
//
// LDS rows are 128 bytes apart, half of its 64 banks; 16-byte piece c of row r lies at place c ^ (r / 2 % 8), so that 16 lanes that read one piece of 16
// rows use every bank once (with r % 8 in its place half of the LDS cycles were conflicts). The copies to LDS write a wave's 1 KB in lane order: the
// exchange is made in the addresses that the lanes read from.
//
// Bound: a step of a 256 x 256 tile has 2048 cycles of products on every SIMD next to 192 KB of LDS reads by eight waves of 128 x 64 and 64 KB of copies (four waves of 128 x 128 read
// 128 KB, but a wave alone on its SIMD leaves it idle at every wait: bf16 8192 x 8192 x 8192 895 us, eight waves 820 = 1.34 PFLOP/s at 1.82 GHz, 71 % of the cycles in products).
// Smaller tiles are bound by LDS (64 x 128: 48 KB of reads for 256 cycles of products) and are for fewer results than fill the chip. fp32 and fp64 are bound by their
// matrix instructions at any size (16 x 16 x 4: 32 and 64 cycles).
#pragma once
#include "cla_device.hpp"

namespace cla {

typedef int mm_i32x4 __attribute__((ext_vector_type(4)));
typedef int mm_i32x16 __attribute__((ext_vector_type(16)));
typedef float mm_f32x4 __attribute__((ext_vector_type(4)));
typedef float mm_f32x16 __attribute__((ext_vector_type(16)));
typedef double mm_f64x2 __attribute__((ext_vector_type(2)));
typedef double mm_f64x4 __attribute__((ext_vector_type(4)));
typedef __bf16 mm_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 mm_f16x8 __attribute__((ext_vector_type(8)));

// What a type's values are computed in: fp32, and fp64 for fp64.
template <class T> struct MmCalc { typedef float type; };
template <> struct MmCalc<double> { typedef double type; };

// An operand type on the matrix cores. FR: rows of a fragment (16 bytes of FR rows in 64 lanes: 64 / FR pieces of the summed index). A lane's results belong to row lane % FR of the rows' operand
// and to the columns mm_col(lane, r) of the other, MmGroup of them next to each other.
template <class E> struct MmOp;
template <> struct MmOp<int8_t> {
	static constexpr int FR = 32;
	typedef int Sum;
	typedef mm_i32x16 Acc;
	typedef mm_i32x4 Acc16;
	static __device__ __forceinline__ void mma(Acc& c, mm_i32x4 a, mm_i32x4 b) { c = __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0); }
	static __device__ __forceinline__ void mma16(Acc16& c, mm_i32x4 a, mm_i32x4 b) { c = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
};
template <> struct MmOp<__bf16> {
	static constexpr int FR = 32;
	typedef float Sum;
	typedef mm_f32x16 Acc;
	typedef mm_f32x4 Acc16;
	static __device__ __forceinline__ void mma(Acc& c, mm_i32x4 a, mm_i32x4 b) {
		c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(mm_bf16x8, a), __builtin_bit_cast(mm_bf16x8, b), c, 0, 0, 0);
	}
	static __device__ __forceinline__ void mma16(Acc16& c, mm_i32x4 a, mm_i32x4 b) {
		c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mm_bf16x8, a), __builtin_bit_cast(mm_bf16x8, b), c, 0, 0, 0);
	}
};
template <> struct MmOp<_Float16> {
	static constexpr int FR = 32;
	typedef float Sum;
	typedef mm_f32x16 Acc;
	typedef mm_f32x4 Acc16;
	static __device__ __forceinline__ void mma(Acc& c, mm_i32x4 a, mm_i32x4 b) {
		c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(mm_f16x8, a), __builtin_bit_cast(mm_f16x8, b), c, 0, 0, 0);
	}
	static __device__ __forceinline__ void mma16(Acc16& c, mm_i32x4 a, mm_i32x4 b) {
		c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(mm_f16x8, a), __builtin_bit_cast(mm_f16x8, b), c, 0, 0, 0);
	}
};
template <> struct MmOp<float> { // (16 rows: the same rate, and tiles half as large)
	static constexpr int FR = 16;
	typedef float Sum;
	typedef mm_f32x4 Acc;
	typedef mm_f32x4 Acc16;
	static __device__ __forceinline__ void mma(Acc& c, mm_i32x4 a, mm_i32x4 b) {
		const mm_f32x4 x = __builtin_bit_cast(mm_f32x4, a), y = __builtin_bit_cast(mm_f32x4, b);
#pragma unroll
		for(int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], c, 0, 0, 0);
	}
	static __device__ __forceinline__ void mma16(Acc16& c, mm_i32x4 a, mm_i32x4 b) { mma(c, a, b); }
};
template <> struct MmOp<double> {
	static constexpr int FR = 16;
	typedef double Sum;
	typedef mm_f64x4 Acc;
	typedef mm_f64x4 Acc16;
	static __device__ __forceinline__ void mma(Acc& c, mm_i32x4 a, mm_i32x4 b) {
		const mm_f64x2 x = __builtin_bit_cast(mm_f64x2, a), y = __builtin_bit_cast(mm_f64x2, b);
#pragma unroll
		for(int i = 0; i < 2; i++) c = __builtin_amdgcn_mfma_f64_16x16x4f64(x[i], y[i], c, 0, 0, 0);
	}
	static __device__ __forceinline__ void mma16(Acc16& c, mm_i32x4 a, mm_i32x4 b) { mma(c, a, b); }
};

// The column (of a fragment) that result r of this lane belongs to; its row is lane % FR. Results come in groups of MmGroup neighbouring columns.
template <class E>
__device__ __forceinline__ int mm_col16(int lane, int r) { return std::is_same<E, double>::value ? 4 * r + (lane >> 4) : 4 * (lane >> 4) + r; }
template <class E>
__device__ __forceinline__ int mm_col(int lane, int r) { return MmOp<E>::FR == 32 ? 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3) : mm_col16<E>(lane, r); }
template <class E> struct MmGroup { static constexpr int value = std::is_same<E, double>::value ? 1 : 4; };

// exp and 1 / x for values that are rounded to T: 16-bit results take the instructions for 2^x and 1 / x (relative errors: 2^-22 of either, and 2^-23 |x| of the exponential, from its
// argument's rounding), fp32 and fp64 the full functions.
template <class T> struct MmMath {
	typedef typename MmCalc<T>::type C;
	static __device__ __forceinline__ C exp_of(C x) { return exp(x); }
	static __device__ __forceinline__ C inverse(C x) { return C(1) / x; }
};
template <> struct MmMath<float> {
	static __device__ __forceinline__ float exp_of(float x) { return expf(x); }
	static __device__ __forceinline__ float inverse(float x) { return 1.0f / x; }
};
struct MmMathShort {
	static __device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(1.44269504088896341f * x); }
	static __device__ __forceinline__ float inverse(float x) { return __builtin_amdgcn_rcpf(x); }
};
template <> struct MmMath<__bf16> : MmMathShort {};
template <> struct MmMath<_Float16> : MmMathShort {};
__device__ __forceinline__ float mm_erfc(float x) { return erfcf(x); }
__device__ __forceinline__ double mm_erfc(double x) { return erfc(x); }

// The logistic function, and of both signs of x: 1 - l(x) is l(-x), which a difference would lose where it is small. (exp overflows to infinity, 1 / infinity is 0: the limit.)
template <class T, class C>
__device__ __forceinline__ C mm_logistic(C x) { return MmMath<T>::inverse(C(1) + MmMath<T>::exp_of(-x)); }
template <class T, class C>
__device__ __forceinline__ void mm_logistics(C x, C& of, C& minus) {
	const C e = MmMath<T>::exp_of(-fabs(x)), l = MmMath<T>::inverse(C(1) + e);
	of = x < C(0) ? e * l : l; minus = x < C(0) ? l : e * l;
}

// The activation of a gated unit (act: enum cla_act) and its derivative, for results of type T. Each in a form that keeps its digits where it is small: Phi(x) = erfc(-x / sqrt 2) / 2,
// (1 + tanh a) / 2 = l(2 a). (As 1 + erf, 1 + tanh and l (1 - l): gelu(-5) 4 %, its approximation there 30 %, the logistic function's derivative at 12 1 % off in fp32.)
enum : int { ACT_SIGMOID = 0, ACT_SILU = 1, ACT_GELU = 2, ACT_GELU_TANH = 3, ACT_RELU = 4, ACT_NONE = 5 };
template <class T, class C>
__device__ __forceinline__ C mm_act(C x, int act) {
	switch(act) { // (uniform)
		case ACT_SIGMOID: return mm_logistic<T>(x);
		case ACT_SILU: return x * mm_logistic<T>(x);
		case ACT_GELU: return C(0.5) * x * mm_erfc(x * C(-0.70710678118654752440));
		case ACT_GELU_TANH: return x * mm_logistic<T>(C(1.59576912160573071176) * (x + C(0.044715) * x * x * x));
		case ACT_RELU: return x < C(0) ? C(0) : x; // (a NaN stays one)
		default: return x;
	}
}
// value and derivative
template <class T, class C>
__device__ __forceinline__ void mm_act_both(C x, int act, C& value, C& slope) {
	C l, m; // l(.), l(-.)
	switch(act) {
		case ACT_SIGMOID: { mm_logistics<T>(x, l, m); value = l; slope = l * m; break; }
		case ACT_SILU: { mm_logistics<T>(x, l, m); value = x * l; slope = l * (C(1) + x * m); break; }
		case ACT_GELU: {
			const C p = C(0.5) * mm_erfc(x * C(-0.70710678118654752440));
			value = x * p; slope = p + x * MmMath<T>::exp_of(C(-0.5) * x * x) * C(0.39894228040143267794);
			break;
		}
		case ACT_GELU_TANH: {
			mm_logistics<T>(C(1.59576912160573071176) * (x + C(0.044715) * x * x * x), l, m);
			const C w = l * m; // (0 long before x * x leaves the range)
			value = x * l;
			slope = w > C(0) ? l + x * w * C(1.59576912160573071176) * (C(1) + C(0.134145) * x * x) : l;
			break;
		}
		case ACT_RELU: { value = x < C(0) ? C(0) : x; slope = x > C(0) ? C(1) : C(0); break; }
		default: { value = x; slope = C(1); break; }
	}
}

// n consecutive values as one access
template <class T, int N> struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) MmPack { T x[N]; };
// ... to or from an address that need not be a multiple of their size. (As whole words: a copy of values becomes an access for each.)
template <int BYTES> struct MmWord { typedef mm_i32x4 type; };
template <> struct MmWord<8> { typedef uint64_t type; };
template <> struct MmWord<4> { typedef uint32_t type; };
template <> struct MmWord<2> { typedef uint16_t type; };
template <class P>
__device__ __forceinline__ void mm_put(void* to, const P& p) {
	const typename MmWord<sizeof(P)>::type w = __builtin_bit_cast(typename MmWord<sizeof(P)>::type, p);
	__builtin_memcpy(to, &w, sizeof(P));
}
template <class P>
__device__ __forceinline__ P mm_get(const void* from) {
	typename MmWord<sizeof(P)>::type w;
	__builtin_memcpy(&w, from, sizeof(P));
	return __builtin_bit_cast(P, w);
}

// 16 bytes of elements of ES bytes from any address of their alignment, `left` bytes of the row from there on: what lies behind the row is 0. PARTIAL: rows
// need not end at multiples of 16 bytes.
template <int ES, bool PARTIAL = true>
__device__ __forceinline__ mm_i32x4 mm_load16(const char* p, int64_t left) {
	mm_i32x4 v = {0, 0, 0, 0};
	if(left >= 16) __builtin_memcpy(&v, p, 16);
	if(PARTIAL && left > 0 && left < 16) { // (rare: behind a branch of its own, so that a lane's next loads do not wait for it)
		if(ES == 8) { // (one of two)
			uint64_t x;
			__builtin_memcpy(&x, p, 8);
			v[0] = (int) (uint32_t) x; v[1] = (int) (x >> 32);
		}
		else if(ES == 4) {
#pragma unroll
			for(int i = 0; i < 3; i++)
				if(4 * i < left) { uint32_t x; __builtin_memcpy(&x, p + 4 * i, 4); v[i] = (int) x; }
		}
		else if(ES == 2) {
#pragma unroll
			for(int i = 0; i < 7; i++)
				if(2 * i < left) { uint16_t x; __builtin_memcpy(&x, p + 2 * i, 2); v[i >> 1] |= (int) ((uint32_t) x << (16 * (i & 1))); }
		}
		else {
#pragma unroll
			for(int i = 0; i < 15; i++)
				if(i < left) v[i >> 2] |= (int) ((uint32_t) (uint8_t) p[i] << (8 * (i & 3)));
		}
	}
	return v;
}

struct MmArgs {
	const char* rows;         // M rows, ldRows bytes apart
	const char* cols;         // N columns (gated: the gate's N, then the other projection's N), ldCols bytes apart
	int64_t ldRows, ldCols;
	int64_t zRows, zCols;     // bytes between the operands of successive parts of the summed index (split)
	int64_t M;
	int32_t N;                // columns of the output
	int64_t K, kPart;         // bytes of the summed index in all and of a part
	int32_t tilesM, tilesN, parts;
};

constexpr unsigned MM_OUT = 0x70000000u; // an offset behind every operand's end: such a load is answered with zeros
constexpr int64_t MM_MAX_LD = 4 << 20;   // bytes: a tile's offsets (256 rows) stay within 2^30

// E: operands, TM x TN: rows and columns (gated: TN / 2 columns of either projection) of a tile, WM x WN waves, DEPTH steps in LDS. DIRECT: operands whose
// rows begin and end at multiples of 4 bytes go from global memory to LDS without registers, DEPTH - 1 steps ahead (what a row's last 16 bytes hold of the next
// row is cleared in LDS); others are loaded a step ahead into registers.
template <class E_, int TM_, int TN_, int WM_, int WN_, int DEPTH_, bool GATED_, bool DIRECT_> struct MmShape {
	typedef E_ E;
	static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, DEPTH = DIRECT_ ? DEPTH_ : 2, THREADS = 64 * WM * WN;
	static constexpr bool GATED = GATED_, DIRECT = DIRECT_;
	static constexpr int NF = TN / WN / MmOp<E>::FR;
	// operands may end inside 16 bytes: not in 8 bits, whose weights are padded, nor on the largest tile, which the question alone makes 2 % slower (gated unit of 4096 x 4096 into 2 x 12288 in bf16 686 and 673 us)
	static constexpr bool ENDS = sizeof(E) > 1 && TM * TN < 256 * 256;
	template <class Epi> static constexpr size_t lds() { // (the epilogue takes over what the steps have used)
		const size_t steps = (size_t) DEPTH * (TM + TN) * 128, out = (size_t) WM * WN * Epi::template region<E, NF, GATED>();
		return steps > out ? steps : out;
	}
};

#ifdef __HIP_DEVICE_COMPILE__ // (the host pass knows no buffer descriptors)
template <class Shape, class Epi>
__device__ __forceinline__ void mm_tile(const MmArgs& A, const Epi& epi, unsigned block, unsigned blocks, char* mm_smem) {
	typedef typename Shape::E E;
	typedef MmOp<E> Op;
	constexpr int TM = Shape::TM, TN = Shape::TN, WM = Shape::WM, WN = Shape::WN, DEPTH = Shape::DEPTH;
	constexpr bool GATED = Shape::GATED, DIRECT = Shape::DIRECT;
	constexpr int FR = Op::FR, NW = WM * WN, PIECES = 64 / FR, SUB = 8 / PIECES;
	constexpr int SM = TM / WM, SN = TN / WN, MF = SM / FR, NF = SN / FR;
	constexpr int LM = TM / 8 / NW, LN = TN / 8 / NW, BUF = (TM + TN) * 128;
	constexpr bool ENDS = Shape::DIRECT && Shape::ENDS;
	static_assert(SUB % 2 == 0 && LM * 8 * NW == TM && LN * 8 * NW == TN && (!GATED || NF % 2 == 0) && (DEPTH & (DEPTH - 1)) == 0, "tile");
	const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);

	// Tiles go to the XCDs in runs (their L2s see neighbours), within a run 8 row tiles share each of the column tiles.
	int tm, tn, part;
	{
		const unsigned xcd = block % 8, at = block / 8, q = blocks / 8, rest = blocks % 8;
		unsigned t = xcd * q + min(xcd, rest) + at;
		const unsigned per = (unsigned) A.tilesM * (unsigned) A.tilesN;
		part = (int) (t / per);
		t -= (unsigned) part * per;
		const unsigned width = 8u * (unsigned) A.tilesN, group = t / width, in = t - group * width, gm = min((unsigned) A.tilesM - group * 8u, 8u);
		tm = (int) (group * 8u + in % gm);
		tn = (int) (in / gm);
	}
	const int64_t m0 = (int64_t) tm * TM;
	const int n0 = tn * (GATED ? TN / 2 : TN);
	const int64_t left = A.K - (int64_t) part * A.kPart, K = left < A.kPart ? left : A.kPart; // bytes of this part
	const int nk = (int) ((K + 127) >> 7);
	const int rowsIn = (int) min(A.M - m0, (int64_t) TM), colsIn = min(A.N - n0, GATED ? TN / 2 : TN);
	const char* const pRows = A.rows + part * A.zRows + m0 * A.ldRows;
	const char* const pCols = A.cols + part * A.zCols + (int64_t) n0 * A.ldCols;
	const char* const pUp = GATED ? pCols + (int64_t) A.N * A.ldCols : pCols;
	const int ldR = (int) A.ldRows, ldC = (int) A.ldCols; // (at most MM_MAX_LD, or 2^31 - 1 where offsets are not held in 32 bits)

	// a wave takes every NW-th 8 rows of the tile; lane: row lane / 8 of them, the piece of the step that belongs at place lane % 8
	static_assert(NW % 2 == 0, "a wave's rows / 2 are alike modulo 8");
	const int lr = lane >> 3, piece = ((lane & 7) ^ (((wave & 1) << 2) + (lr >> 1))) * 16;
	auto col_half = [&](int i) { return GATED ? ((i * 8) / FR) & 1 : 0; };                     // gate's or the other projection's
	auto col_row = [&](int i) { return GATED ? ((i * 8) / (2 * FR)) * FR + (i * 8) % FR : i * 8; }; // first of 8 columns
	__amdgpu_buffer_rsrc_t rRows, rCols, rUp;
	if(DIRECT) {
		// (up to the last row's last value: 4 bytes at a time, what lies behind is answered with zeros)
		const int endR = (rowsIn - 1) * ldR + (int) K, endC = (colsIn - 1) * ldC + (int) K;
		rRows = __builtin_amdgcn_make_buffer_rsrc((void*) pRows, 0, endR, 0x00020000);
		rCols = __builtin_amdgcn_make_buffer_rsrc((void*) pCols, 0, endC, 0x00020000);
		if(GATED) rUp = __builtin_amdgcn_make_buffer_rsrc((void*) pUp, 0, endC, 0x00020000);
	}
	mm_i32x4 hold[DIRECT ? 1 : LM + LN];
	auto issue = [&](int t, int which) { // step t's rows (1), columns (2): on their way to LDS (buffer t % DEPTH), or into registers
		const int k = t * 128;
		if(DIRECT) {
			char* const to = mm_smem + (t & (DEPTH - 1)) * BUF;
			const bool out = k + piece >= K;
			// (ENDS: the step's place is part of the lane's offset, since the descriptor's end is not held against the scalar one and a last row's last 16 bytes may begin in
			// front of it; elsewhere it is the scalar one: 8-bit gated unit of 4096 x 4096 into 2 x 12288 390 and 385 us, gradients at 2 x 8192 in bf16 1489 and 1464)
			const int kv = ENDS ? k : 0, ks = ENDS ? 0 : k;
			const unsigned vr = out ? MM_OUT : (unsigned) (lr * ldR + piece + kv), vc = out ? MM_OUT : (unsigned) (lr * ldC + piece + kv);
#pragma unroll
			for(int j = 0; j < (which & 1 ? LM : 0); j++) {
				const int i = j * NW + wave;
				__builtin_amdgcn_raw_ptr_buffer_load_lds(rRows, (__attribute__((address_space(3))) void*) (to + i * 1024), 16, (int) (vr + (unsigned) (i * 8 * ldR)), ks, 0, 0);
			}
#pragma unroll
			for(int j = 0; j < (which & 2 ? LN : 0); j++) {
				const int i = j * NW + wave;
				__builtin_amdgcn_raw_ptr_buffer_load_lds(col_half(i) ? rUp : rCols, (__attribute__((address_space(3))) void*) (to + TM * 128 + i * 1024), 16,
					(int) (vc + (unsigned) (col_row(i) * ldC)), ks, 0, 0);
			}
		}
		else {
#pragma unroll
			for(int j = 0; j < LM; j++) {
				const int r = (j * NW + wave) * 8 + lr;
				hold[j] = mm_load16<sizeof(E)>(pRows + (int64_t) r * ldR + k + piece, r < rowsIn ? K - k - piece : 0);
			}
#pragma unroll
			for(int j = 0; j < LN; j++) {
				const int i = j * NW + wave, c = col_row(i) + lr;
				hold[LM + j] = mm_load16<sizeof(E)>((col_half(i) ? pUp : pCols) + (int64_t) c * ldC + k + piece, c < colsIn ? K - k - piece : 0);
			}
		}
	};
	auto clean = [&](int t) { // the last step, if the operands end inside 16 bytes: zeros behind their end (each lane in what it has copied)
		const int valid = (int) K - t * 128 - piece;
		if(!ENDS || valid <= 0 || valid >= 16) return;
		char* const to = mm_smem + (t & (DEPTH - 1)) * BUF + lane * 16;
#pragma unroll
		for(int j = 0; j < LM + LN; j++) {
			char* const at = to + (j < LM ? (j * NW + wave) * 1024 : TM * 128 + ((j - LM) * NW + wave) * 1024);
#pragma unroll
			for(int b = 4; b < 16; b += 4)
				if(b >= valid) *(int*) (at + b) = 0;
		}
	};
	auto put = [&](int t) { // the registers' step into LDS
		char* const to = mm_smem + (t & 1) * BUF + lane * 16;
#pragma unroll
		for(int j = 0; j < LM; j++) *(mm_i32x4*) (to + (j * NW + wave) * 1024) = hold[j];
#pragma unroll
		for(int j = 0; j < LN; j++) *(mm_i32x4*) (to + TM * 128 + (j * NW + wave) * 1024) = hold[LM + j];
	};

	const int wm = wave % WM, wn = wave / WM;
	constexpr int H = GATED ? 2 : 1;
	const int fragments = H * ((A.N - n0 - wn * (SN / H) + FR - 1) / FR); // of the wave's columns that are there
	typename Op::Acc acc[NF][MF];
#pragma unroll
	for(int i = 0; i < NF; i++)
#pragma unroll
		for(int j = 0; j < MF; j++)
#pragma unroll
			for(int r = 0; r < FR * FR / 64; r++) acc[i][j][r] = 0;
	mm_i32x4 fc[2][NF], fr[2][MF];
	const int fl = (lane % FR) * 128;
	auto read = [&](int set, int t, int s) {
		const char* const from = mm_smem + (t & (DEPTH - 1)) * BUF + fl + (((s * PIECES + lane / FR) ^ ((lane % FR >> 1) & 7)) << 4);
#pragma unroll
		for(int j = 0; j < MF; j++) fr[set][j] = *(const mm_i32x4*) (from + (wm * SM + j * FR) * 128);
#pragma unroll
		for(int i = 0; i < NF; i++) fc[set][i] = *(const mm_i32x4*) (from + (TM + wn * SN + i * FR) * 128);
	};
	auto barrier = [&]() {
		asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
		__builtin_amdgcn_s_barrier();
		asm volatile("" ::: "memory");
	};

	if(nk > 0) {
		if(DIRECT) {
#pragma unroll
			for(int t = 0; t < DEPTH; t++)
				if(t < nk) issue(t, 3);
			if(nk >= DEPTH) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((DEPTH - 1) * (LM + LN)) : "memory");
			else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
			if(ENDS && nk == 1) clean(0);
		}
		else {
			issue(0, 3);
			put(0);
		}
		barrier();
		read(0, 0, 0);
	}
	for(int t = 0; t < nk; t++) {
		if(!DIRECT && t + 1 < nk) issue(t + 1, 3);
#pragma unroll
		for(int s = 0; s < SUB; s++) {
			// (a step's columns follow its rows a part of a step later: a wave cannot issue anything else while its copies wait in line)
			if(DIRECT && s == 0 && t > 0 && t + DEPTH - 1 < nk) issue(t + DEPTH - 1, 2);
			if(s + 1 < SUB) read((s + 1) & 1, t, s + 1);
			else if(t + 1 < nk) {
				// everything of step t has been read; of the steps requested since, step t + 1 has to be there
				if(DIRECT) {
					if(DEPTH > 2 && t + DEPTH - 1 < nk) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((DEPTH - 2) * (LM + LN)) : "memory");
					else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
					if(ENDS && t + 2 == nk) clean(t + 1);
					barrier();
					if(t + DEPTH < nk) issue(t + DEPTH, 1);
				}
				else {
					put(t + 1); // (its buffer was last read in step t - 1)
					barrier();
				}
				read(0, t + 1, 0);
			}
#pragma unroll
			for(int i = 0; i < NF; i++)
#pragma unroll
				for(int j = 0; j < MF; j++) {
					if(sizeof(E) > 2 && ((s > 0 && t * 128 + s * PIECES * 16 >= K) || i >= fragments)) continue; // (what lies behind the operands' ends: uniform)
					Op::mma(acc[i][j], fc[s & 1][i], fr[s & 1][j]);
				}
			if(sizeof(E) <= 2) { // the next reads and copies between the products, not in front of them
#pragma unroll
				for(int q = 0; q < NF * MF; q++) {
					__builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                   // a product
					if(q < NF + MF) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);   // an LDS read
					if(q < LM) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);        // a copy
				}
			}
		}
	}
	barrier(); // LDS is the epilogue's
	epi.template run<E, MF, NF, GATED>(acc, mm_smem + wave * Epi::template region<E, NF, GATED>(), m0 + wm * SM, n0 + wn * (GATED ? SN / 2 : SN), A.M, A.N, part, tm * WM + wm, lane);
}
#endif

constexpr int MM_WAVES = 2; // waves to a SIMD that the registers leave room for

template <class Shape, class Epi>
__global__ __launch_bounds__(Shape::THREADS, MM_WAVES) void k_mm(MmArgs A, Epi epi) {
#ifdef __HIP_DEVICE_COMPILE__
	extern __shared__ __attribute__((aligned(16))) char mm_smem[];
	mm_tile<Shape>(A, epi, blockIdx.x, gridDim.x, mm_smem);
#endif
}

// A product and other work in one launch: blocks below `blocks` take its tiles, `more` gets the others, counted from 0.
template <class Shape, class Epi, class More>
__global__ __launch_bounds__(Shape::THREADS, MM_WAVES) void k_mm_and(MmArgs A, Epi epi, unsigned blocks, More more) {
#ifdef __HIP_DEVICE_COMPILE__
	extern __shared__ __attribute__((aligned(16))) char mm_smem[];
	if(blockIdx.x < blocks) mm_tile<Shape>(A, epi, blockIdx.x, blocks, mm_smem);
	else more.run(blockIdx.x - blocks, mm_smem);
#endif
}

// Two products and other work in one launch.
template <class Shape, class EpiA, class EpiB, class More>
__global__ __launch_bounds__(Shape::THREADS, MM_WAVES) void k_mm_two(MmArgs A, EpiA epiA, unsigned blocksA, MmArgs B, EpiB epiB, unsigned blocksB, More more) {
#ifdef __HIP_DEVICE_COMPILE__
	extern __shared__ __attribute__((aligned(16))) char mm_smem[];
	const unsigned b = blockIdx.x;
	if(b < blocksA) mm_tile<Shape>(A, epiA, b, blocksA, mm_smem);
	else if(b - blocksA < blocksB) mm_tile<Shape>(B, epiB, b - blocksA, blocksB, mm_smem);
	else more.run(b - blocksA - blocksB, mm_smem);
#endif
}

// The same for few rows (up to 16 MR): columns are a stream of bytes that is read once, from global memory straight into the matrix operand. A block
// takes 16 columns (gated: of either projection), its waves take turns of the summed index and add their sums up in LDS, in the order of the waves.
// Lane: column (and row) lane % 16, 16 bytes from 16 (lane / 16) on of every 64. Rows that are not there are zeros. A turn's columns are requested two turns
// ahead, the first ones in front of `before` (what has to be done before rowOf gives rows).
constexpr int MMF_WAVES = 8, MMF_UNROLL = 4;
// Whether that is faster than tiles: up to 16 rows, or so few results that tiles would leave most of the chip idle. In sixteens of rows times sixteens of columns, us
// here / on tiles, K = 4096: bf16 gated 32 x 4096 (512) 19 / 30, 32 x 8192 (1024) 37 / 31, 64 x 4096 (1024) 26 / 31, 64 x 8192 (2048) 52 / 31; 8-bit 32 x 8192 (1024) 13 / 16,
// 32 x 12288 (1536) 20 / 17, 37 x 7681 of K = 5001 (1443) 18 / 21, 64 x 4096 (1024) 12 / 16, 64 x 8192 (2048) 23 / 17; fp32 256 x 2048 (2048) 144 / 148, fp64 246 / 286, 512 x 2048 (4096) 280 / 154 and 487 / 288.
template <class E>
static inline bool mm_few_suits(int64_t m, int64_t n, int cus) {
	return m <= 16 || (m + 15) / 16 * ((n + 15) / 16) <= (sizeof(E) == 1 ? 6 : sizeof(E) == 2 ? 4 : 8) * (int64_t) cus;
}
// How many rows (in sixteens) a block takes: up to 64, as few as it needs to give every CU one (48 where that holds all: 37 rows, us
// with 48 / without: bf16 gated 4096 into 2 x 4096 21 / 30, into 2 x 4864 37 / 40, fp32 62 / 83 and 107 / 111, 8-bit 5001 into 7681 22 / 26, 8-bit gated 4096 into 2 x 4096 16 / 21).
static inline int mm_few_rows(int64_t m, int64_t n, int cus) {
	for(int r = 4; r > 1; r--)
		if(m > 16 * (r - 1) && (r != 3 || m <= 48) && (m + 16 * r - 1) / (16 * r) * ((n + 15) / 16) >= cus) return r;
	return 1;
}
template <class E, bool GATED, int MR, class Rows, class Before>
__device__ __forceinline__ void mm_few(const char* cols, int64_t ldCols, int n0, int N, int64_t K, const Rows& rowOf, const Before& before,
	typename MmOp<E>::Acc16 (&acc)[GATED ? 2 : 1][MR], int wave, int lane) {
	typedef MmOp<E> Op;
	constexpr int H = GATED ? 2 : 1, U = MMF_UNROLL;
	constexpr int64_t TURN = 64 * U, STEP = MMF_WAVES * TURN;
	const int l16 = lane & 15;
	const int64_t at = (lane >> 4) * 16;
	const int c = min(n0 + l16, N - 1);
	const char* const p[2] = {cols + (int64_t) c * ldCols + at, cols + ((int64_t) c + (GATED ? N : 0)) * ldCols + at};
	mm_i32x4 w[2][H][U];
	auto load = [&](int set, int64_t k) { // (8-bit weights are held in whole 128 bytes)
#pragma unroll
		for(int u = 0; u < U; u++)
#pragma unroll
			for(int h = 0; h < H; h++) w[set][h][u] = mm_load16<sizeof(E), (sizeof(E) > 1)>(p[h] + k + u * 64, K - (k + u * 64 + at));
	};
	auto multiply = [&](int set, int64_t k) {
		mm_i32x4 y[MR][U];
#pragma unroll
		for(int u = 0; u < U; u++)
#pragma unroll
			for(int j = 0; j < MR; j++) y[j][u] = rowOf(16 * j + l16, k + u * 64 + at, K - (k + u * 64 + at));
#pragma unroll
		for(int u = 0; u < U; u++)
#pragma unroll
			for(int h = 0; h < H; h++)
#pragma unroll
				for(int j = 0; j < MR; j++) Op::mma16(acc[h][j], w[set][h][u], y[j][u]);
	};
#pragma unroll
	for(int h = 0; h < H; h++)
#pragma unroll
		for(int j = 0; j < MR; j++) acc[h][j] = typename Op::Acc16{0, 0, 0, 0};
	int64_t k = wave * TURN;
	if(k < K) load(0, k);
	if(k + STEP < K) load(1, k + STEP);
	before();
	while(k < K) { // (uniform)
		multiply(0, k);
		if(k + 2 * STEP < K) load(0, k + 2 * STEP);
		k += STEP;
		if(k >= K) break;
		multiply(1, k);
		if(k + 2 * STEP < K) load(1, k + 2 * STEP);
		k += STEP;
	}
}

} // namespace cla
