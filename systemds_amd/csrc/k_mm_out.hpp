// What a tile of k_mm.hpp does with its sums: a wave passes them through a region of LDS of its own, fragment of rows by fragment, so that everything
// that follows (scales, biases, activations, stores) is done on neighbouring columns of a row, 16 bytes of the output at a time.
#pragma once
#include "k_mm.hpp"

namespace cla {

__device__ __forceinline__ void mm_wave_sync() { // what the wave's lanes wrote to LDS is there for its other lanes
	__builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
	__builtin_amdgcn_wave_barrier();
}

// The region: [half][row of the fragment][column], the halves of a gated unit apart.
template <class E, int NF, bool GATED> struct MmRegion {
	typedef typename MmOp<E>::Sum Sum;
	static constexpr int FR = MmOp<E>::FR, H = GATED ? 2 : 1, COLS = NF * FR / H, R = FR * FR / 64, W = MmGroup<E>::value;
	static constexpr int PITCH = COLS * (int) sizeof(Sum) + 16, HALF = FR * PITCH, BYTES = H * HALF;
	template <int MF, class Acc>
	static __device__ __forceinline__ void put(char* region, Acc (&acc)[NF][MF], int j, int lane) {
#pragma unroll
		for(int i = 0; i < NF; i++)
#pragma unroll
			for(int r = 0; r < R; r += W) {
				MmPack<Sum, W> p;
#pragma unroll
				for(int v = 0; v < W; v++) p.x[v] = acc[i][j][r + v];
				*(MmPack<Sum, W>*) (region + (i % H) * HALF + (lane % FR) * PITCH + ((i / H) * FR + mm_col<E>(lane, r)) * (int) sizeof(Sum)) = p;
			}
		mm_wave_sync();
	}
	static __device__ __forceinline__ Sum* at(char* region, int half, int row, int col) {
		return (Sum*) (region + half * HALF + row * PITCH + col * (int) sizeof(Sum));
	}
};

// A sum of 8-bit products times its row's and column's scales. In fp32 their product may leave the range though the result does not (a sum of 2^25 with scales of 2^-70 each; a sum of 0 with
// scales of 2^100): in 64 bits then.
template <class C>
__device__ __forceinline__ C mm_scaled_wide(C sum, C s, C t) { return (C) ((double) sum * (double) s * (double) t); }
template <class C>
__device__ __forceinline__ bool mm_scales_fit(C least, C most) { return sizeof(C) == 8 || (least >= C(1.17549435e-38f) && most <= C(3.4028234663852886e38f)); } // (not of a NaN)
template <class C>
__device__ __forceinline__ C mm_scaled(C sum, C s, C t) {
	const C p = s * t, a = fabs(p);
	return mm_scales_fit(a, a) ? sum * p : mm_scaled_wide(sum, s, t);
}

// V values to a row of the output, `cols` of them there: 16 bytes at once wherever the row begins.
template <class T, int V>
__device__ __forceinline__ void mm_store(T* to, const MmPack<T, V>& x, int cols) {
	if(cols >= V) mm_put(to, x);
	else {
#pragma unroll
		for(int v = 0; v < V; v++)
			if(v < cols) to[v] = x.x[v];
	}
}

// A power of two that brings magnitudes up to `most` (a float's bits) below 2^15, and what takes it back: within 2^-113 .. 2^120, so that both are ordinary numbers. 1 for
// a bound that is not finite (what it bounds is not either).
__device__ __forceinline__ float mm_pow2(uint32_t most, bool back) {
	const int e = (int) (most >> 23), k = e >= 255 ? 0 : min(141 - e, 120);
	return __uint_as_float((uint32_t) (127 + (back ? -k : k)) << 23);
}

// The sums, times a scale for each row and column (SCALED: sums of 8-bit products) or what takes back the power of two of each row (POWERS), plus a bias for each column; gated: activation of the
// gate's times the other projection's. Rounded to T once.
template <class T, bool SCALED, bool POWERS = false> struct MmEpiOut {
	const float* sRow;  // (POWERS: the rows' bounds)
	const float* sCol;
	const T* bias;      // null: none
	T* out;
	int64_t ld;         // values
	int32_t act;
	int64_t zOut;       // values between the outputs of the parts of the summed index

	template <class E, int NF, bool GATED> static constexpr int region() { return MmRegion<E, NF, GATED>::BYTES; }
	template <class E, int MF, int NF, bool GATED, class Acc>
	__device__ __forceinline__ void run(Acc& acc, char* region, int64_t m0, int n0, int64_t M, int N, int part, int, int lane) const {
		typedef MmRegion<E, NF, GATED> Reg;
		typedef typename MmCalc<T>::type C;
		constexpr int FR = Reg::FR, H = Reg::H, V = 16 / (int) sizeof(T), PER = Reg::COLS / V;
		static_assert(Reg::COLS % V == 0, "a row of the region is whole stores");
		static_assert(64 % PER == 0 && FR * PER % 64 == 0, "a lane keeps its columns");
		// a lane's columns are the same ones in every row: their scales and biases stay in registers; the scales of the wave's rows are held one by a lane
		const int c = (lane % PER) * V, cols = N - n0 - c;
		C sc[H][V], bi[H][V], least = C(INFINITY), most = C(0); // (magnitudes of the scales that are not 0)
		float sr[(MF * FR + 63) / 64];
#pragma unroll
		for(int h = 0; h < H; h++)
#pragma unroll
			for(int v = 0; v < V; v++) {
				const int col = min(n0 + c + v, N - 1) + h * N;
				sc[h][v] = SCALED ? (C) sCol[col] : C(1);
				bi[h][v] = bias ? (C) bias[col] : C(0);
				if(SCALED) {
					const C a = fabs(sc[h][v]);
					least = a > C(0) ? fmin(least, a) : least; most = fmax(most, a);
				}
			}
#pragma unroll
		for(int i = 0; i < (MF * FR + 63) / 64; i++) {
			sr[i] = SCALED || POWERS ? sRow[min(m0 + i * 64 + lane, M - 1)] : 1.0f;
			if(POWERS) sr[i] = mm_pow2(__float_as_uint(sr[i]), true);
		}
		auto rows = [&](auto wide) {
#pragma unroll
			for(int j = 0; j < MF; j++) {
				Reg::template put<MF>(region, acc, j, lane);
				const int64_t row0 = m0 + j * FR;
#pragma unroll 1
				for(int r0 = 0; r0 < FR; r0 += 64 / PER) {
					const int r = r0 + lane / PER;
					const C s = SCALED || POWERS ? (C) __shfl(sr[j * FR / 64], (j * FR + r) & 63, 64) : C(1);
					MmPack<T, V> x;
#pragma unroll
					for(int v = 0; v < V; v++) {
						C y[H];
#pragma unroll
						for(int h = 0; h < H; h++) {
							y[h] = (C) Reg::at(region, h, r, c)[v];
							if(SCALED) y[h] = decltype(wide)::value ? mm_scaled_wide(y[h], s, sc[h][v]) : y[h] * (s * sc[h][v]);
							if(POWERS) y[h] *= s;
							y[h] += bi[h][v];
						}
						x.x[v] = (T) (GATED ? mm_act<T>(y[0], act) * y[H - 1] : y[0]);
					}
					if(row0 + r < M && cols > 0) mm_store<T, V>(out + part * zOut + (row0 + r) * ld + n0 + c, x, cols);
				}
				mm_wave_sync();
			}
		};
		if constexpr(SCALED && sizeof(C) == 4) { // (one way for the wave's whole tile: a choice for each row costs 5 % of the 8-bit gated unit)
			C leastS = C(INFINITY), mostS = C(0);
#pragma unroll
			for(int i = 0; i < (MF * FR + 63) / 64; i++) {
				const C a = fabs(sr[i]);
				leastS = a > C(0) ? fmin(leastS, a) : leastS; mostS = fmax(mostS, a);
			}
#pragma unroll
			for(int d = 32; d > 0; d >>= 1) {
				leastS = fmin(leastS, __shfl_xor(leastS, d, 64)); mostS = fmax(mostS, __shfl_xor(mostS, d, 64));
				least = fmin(least, __shfl_xor(least, d, 64)); most = fmax(most, __shfl_xor(most, d, 64));
			}
			if(__builtin_amdgcn_readfirstlane((int) !mm_scales_fit(leastS * least, mostS * most))) {
				rows(std::true_type());
				return;
			}
		}
		rows(std::false_type());
	}
};

// Backward pass of a gated unit: from the projections G, U (the sums) and the incoming gradient D to dG = D U act'(G) and dU = D act(G), rounded to T once.
// They are written twice, by row (P: what dY sums over) and by column (Pt: what dW sums over, rows of the batch in parts of kPart), with zeros where
// either is rounded up to whole 16 bytes; sums over the wave's rows, of the values before that rounding, for the biases' gradient. fp16: a row of P and a column of Pt are multiplied by a power of
// two before they are rounded (by their bounds, see k_gate_bounds), so that no magnitude leaves the type's range; the products take it back.
template <class T> struct MmEpiBack {
	typedef typename MmCalc<T>::type C;
	const T* bias;      // null: none
	const T* D;
	int64_t ldD;
	T* P;               // null: not wanted
	int64_t ldP;        // two halves of ldP / 2 columns, a multiple of 16 bytes each
	T* Pt;              // null: not wanted
	int64_t kPart;      // a multiple of 256
	C* sums;            // null: not wanted; [wave's rows][2 N]
	int32_t act;
	const uint32_t* mostRow; // fp16: bounds of the rows and of the 2 N columns (bits of floats)
	const uint32_t* mostCol;
	static constexpr bool POWERS = std::is_same<T, _Float16>::value;
	__device__ __forceinline__ C row_power(int64_t m) const { return POWERS ? (C) mm_pow2(mostRow[m], false) : C(1); }
	__device__ __forceinline__ C col_power(int c) const { return POWERS ? (C) mm_pow2(mostCol[c], false) : C(1); }

	template <class E, int NF, bool GATED> static constexpr int region() { return MmRegion<E, NF, GATED>::BYTES; }
	template <class E, int MF, int NF, bool GATED, class Acc>
	__device__ __forceinline__ void run(Acc& acc, char* region, int64_t m0, int n0, int64_t M, int N, int, int rowPart, int lane) const {
		typedef MmRegion<E, NF, GATED> Reg;
		constexpr int FR = Reg::FR, COLS = Reg::COLS, V = 16 / (int) sizeof(T), PER = COLS / V, S = (2 * COLS + 63) / 64;
		static_assert(GATED && COLS % V == 0 && FR % V == 0, "two halves, whole stores both ways");
		static_assert(64 % PER == 0 && FR * PER % 64 == 0, "a lane keeps its columns");
		const int c0 = (lane % PER) * V, cols = N - n0, half = (int) (ldP / 2) - n0;
		C sum[S], bg[V], bu[V];
#pragma unroll
		for(int s = 0; s < S; s++) sum[s] = C(0);
#pragma unroll
		for(int v = 0; v < V; v++) {
			const int col = min(n0 + c0 + v, N - 1);
			bg[v] = bias ? (C) bias[col] : C(0);
			bu[v] = bias ? (C) bias[col + N] : C(0);
		}
#pragma unroll
		for(int j = 0; j < MF; j++) {
			Reg::template put<MF>(region, acc, j, lane);
			const int64_t row0 = m0 + j * FR;
#pragma unroll 1
			for(int r0 = 0; r0 < FR; r0 += 64 / PER) {
				const int r = r0 + lane / PER;
				const bool in = row0 + r < M && c0 < cols;
				const T* const d = D + (row0 + r) * ldD + n0 + c0;
				const C by = POWERS && P ? row_power(min(row0 + r, M - 1)) : C(1);
				MmPack<T, V> g, u, dv;
				if(in && c0 + V <= cols) dv = mm_get<MmPack<T, V>>(d);
				else {
#pragma unroll
					for(int v = 0; v < V; v++) dv.x[v] = in && c0 + v < cols ? d[v] : (T) 0.0f;
				}
#pragma unroll
				for(int v = 0; v < V; v++) {
					const C x = *Reg::at(region, 0, r, c0 + v) + bg[v], y = *Reg::at(region, 1, r, c0 + v) + bu[v];
					C value, slope;
					mm_act_both<T>(x, act, value, slope);
					const bool there = in && c0 + v < cols;
					const C dG = there ? (C) dv.x[v] * y * slope : C(0), dU = there ? (C) dv.x[v] * value : C(0);
					*Reg::at(region, 0, r, c0 + v) = dG; *Reg::at(region, 1, r, c0 + v) = dU;
					g.x[v] = (T) (dG * by); u.x[v] = (T) (dU * by);
				}
				if(P && row0 + r < M && c0 < half) {
					T* const to = P + (row0 + r) * ldP + n0 + c0;
					mm_store<T, V>(to, g, V);
					mm_store<T, V>(to + ldP / 2, u, V);
				}
			}
			mm_wave_sync();
			if(sums) {
#pragma unroll
				for(int s = 0; s < S; s++) {
					const int i = s * 64 + lane;
					if(i < 2 * COLS)
						for(int r = 0; r < FR; r++) sum[s] += *Reg::at(region, i / COLS, r, i % COLS);
				}
			}
			if(Pt && row0 < M) {
				const int64_t part = row0 / kPart, at = row0 - part * kPart;
				T* const to = Pt + part * 2 * N * kPart + at;
#pragma unroll 1
				for(int i = lane; i < 2 * COLS * (FR / V); i += 64) {
					const int r = (i % (FR / V)) * V, c = i / (FR / V) % COLS, h = i / (FR / V) / COLS;
					if(c >= cols || row0 + r >= M) continue;
					const C by = col_power(h * N + n0 + c);
					MmPack<T, V> p;
#pragma unroll
					for(int v = 0; v < V; v++) p.x[v] = (T) (*Reg::at(region, h, r + v, c) * by);
					*(MmPack<T, V>*) (to + (int64_t) (h * N + n0 + c) * kPart + r) = p;
				}
			}
			mm_wave_sync();
		}
		if(sums && m0 < M) {
#pragma unroll
			for(int s = 0; s < S; s++) {
				const int i = s * 64 + lane, c = i % COLS;
				if(i < 2 * COLS && c < cols) sums[(int64_t) rowPart * 2 * N + (i / COLS) * N + n0 + c] = sum[s];
			}
		}
	}
};

} // namespace cla
