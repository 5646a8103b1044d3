// Gated units in the operands' own type: what their entry points ask of the kernels.
#pragma once
#include "cla_internal.hpp"

namespace cla {

struct GateCall {
	int32_t act, type;
	const void* Y; int64_t m; int32_t nIn; int64_t ldY;
	const void* W; int64_t ldW;
	const void* bias;
	int32_t nOut;
	void* out; int64_t ldOut;                                  // forward
	const void* D; int64_t ldD;                                // backward: incoming gradient; null outputs are not wanted
	void* dY; int64_t ldDY;
	void* dW; int64_t ldDW;
	void* dB;
	char* ws;
};

// The backward pass's parts and workspace (bytes from its start).
struct GatePlan {
	int64_t half;                       // columns of a half of P, rounded up to 16 bytes
	int64_t kPartY; int32_t partsY;     // dY: bytes of the columns of P summed at a time (a multiple of 128)
	int64_t kPart; int32_t parts;       // dW: rows of the batch summed at a time (a multiple of 256)
	int32_t sumRows, sumJoins;          // dB: partial sums of a wave's or block's rows (at most so many), and of 64 of those
	size_t P, Pt, Wt, Yt, joinsY, joins, sums, sums64;
	size_t normY, normW, mostRow, mostCol; // fp16: norms of the rows of Y and W, bounds of the rows and columns of P
	size_t bytes;
};

GatePlan gate_plan(int type, int64_t m, int nIn, int nOut);
int launch_gate(const GateCall& c, hipStream_t stream);
int launch_gate_backward(const GateCall& c, hipStream_t stream);
// by type (a translation unit each)
template <class T> int gate_forward(const GateCall& c, hipStream_t stream);
template <class T> int gate_backward(const GateCall& c, hipStream_t stream);

} // namespace cla
