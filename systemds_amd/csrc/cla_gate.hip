// Entry points of the gated units (include/cla_hip.h): checks of arguments, the workspace, host forms. The kernels are in k_gate_impl.hpp.
#include "../../include/cla_hip.h"
#include "k_gate.hpp"
#include "cla_layers.hpp"
#include <algorithm>

namespace cla {

// Parts of a sum of `steps` steps of 128 bytes: two tiles for every CU where there are not enough, at least 8 steps each.
static int64_t gate_parts(int64_t rows, int64_t cols, int64_t steps) {
	const int64_t tiles = ((rows + 127) / 128) * ((cols + 127) / 128);
	if(tiles >= g_numCU) return 1;
	return std::max<int64_t>(1, std::min((2 * g_numCU + tiles - 1) / tiles, steps / 8));
}

GatePlan gate_plan(int type, int64_t m, int nIn, int nOut) {
	GatePlan p{};
	const int64_t es = (int64_t) type_bytes(type), calc = type == CLA_F64 ? 8 : 4, F = nOut;
	p.half = (int64_t) up((size_t) F, (size_t) (16 / es));
	const int64_t stepsY = (2 * p.half * es + 127) / 128, partsY = gate_parts(m, nIn, stepsY);
	p.kPartY = (stepsY + partsY - 1) / partsY * 128;
	p.partsY = (int32_t) ((stepsY * 128 + p.kPartY - 1) / p.kPartY);
	const int64_t parts = gate_parts(2 * F, nIn, m * es / 128);
	p.kPart = std::min((int64_t) up((size_t) ((std::max<int64_t>(m, 1) + parts - 1) / parts), 256), ((int64_t) 4 << 20) / es);
	p.parts = (int32_t) std::max<int64_t>(1, (m + p.kPart - 1) / p.kPart);
	p.sumRows = (int32_t) ((m + 15) / 16);
	p.sumJoins = (p.sumRows + 63) / 64;
	size_t at = 0;
	auto take = [&](int64_t bytes) { const size_t from = at; at += up((size_t) bytes, 256); return from; };
	p.P = take(m * 2 * p.half * es);
	p.Pt = take((int64_t) p.parts * 2 * F * p.kPart * es);
	p.Wt = take(nIn * 2 * p.half * es);
	p.Yt = take((int64_t) p.parts * nIn * p.kPart * es);
	p.joinsY = take(p.partsY > 1 ? (int64_t) p.partsY * m * nIn * calc : 0);
	p.joins = take(p.parts > 1 ? (int64_t) p.parts * 2 * F * nIn * calc : 0);
	p.sums = take((int64_t) p.sumRows * 2 * F * calc);
	p.sums64 = take((int64_t) p.sumJoins * 2 * F * calc);
	if(type == CLA_F16) {
		p.normY = take(m * 4);
		p.normW = take(2 * F * 4);
		p.mostRow = take(m * 4);
		p.mostCol = take(2 * F * 4);
	}
	p.bytes = at;
	return p;
}

static int launch_rows(const GateCall& c, hipStream_t stream) {
	switch(c.type) {
		case CLA_F64: return gate_forward<double>(c, stream);
		case CLA_F32: return gate_forward<float>(c, stream);
		case CLA_BF16: return gate_forward<__bf16>(c, stream);
		default: return gate_forward<_Float16>(c, stream);
	}
}

int launch_gate(const GateCall& c, hipStream_t stream) {
	const int64_t es = (int64_t) type_bytes(c.type), rows = rows_of_a_launch(64, 64, 2 * (int64_t) c.nOut); // (tiles of the smallest shape)
	for(int64_t r = 0; r < c.m; r += rows) {
		GateCall part = c;
		part.m = std::min(c.m - r, rows);
		part.Y = (const char*) c.Y + r * c.ldY * es;
		part.out = (char*) c.out + r * c.ldOut * es;
		if(const int rc = launch_rows(part, stream)) return rc;
	}
	return 0;
}

int launch_gate_backward(const GateCall& c, hipStream_t stream) {
	switch(c.type) {
		case CLA_F64: return gate_backward<double>(c, stream);
		case CLA_F32: return gate_backward<float>(c, stream);
		case CLA_BF16: return gate_backward<__bf16>(c, stream);
		default: return gate_backward<_Float16>(c, stream);
	}
}

// Sizes whose bytes the kernels' offsets and the workspace's hold.
static int check_sizes(const char* what, int type, int64_t m, int nIn, int nOut) {
	int rc;
	if((rc = check_type(what, type)) || (rc = check_rows(what, m))) return rc;
	if(nIn <= 0 || nOut <= 0) { set_error("%s: weights of %d x %d", what, nIn, nOut); return -CLA_ERR_INVALID; }
	const int64_t es = (int64_t) type_bytes(type);
	if(nIn > ((int64_t) 4 << 20) / es || nOut > ((int64_t) 1 << 20) / es) { // 4 MiB a row of Y, 1 MiB a row of the output
		set_error("%s: %d values a row of Y (at most %lld) and %d a row of the output (at most %lld)", what, nIn, (long long) (((int64_t) 4 << 20) / es), nOut,
			(long long) (((int64_t) 1 << 20) / es));
		return -CLA_ERR_UNSUPPORTED;
	}
	return 0;
}

static int check_operands(const char* what, const GateCall& c) {
	int rc;
	if((rc = check_sizes(what, c.type, c.m, c.nIn, c.nOut)) || (rc = check_act(what, c.act))) return rc;
	const size_t es = type_bytes(c.type);
	if(((uintptr_t) c.bias & (es - 1)) != 0) { set_error("%s: bias is not aligned", what); return -CLA_ERR_INVALID; }
	if((rc = check_operand(what, "W", c.W, 2 * (int64_t) c.nOut, c.nIn, c.ldW, es, es))) return rc;
	if(c.m > 0 && (rc = check_operand(what, "Y", c.Y, c.m, c.nIn, c.ldY, es, es))) return rc;
	if(c.ldW * (int64_t) es > 0x7fffffffLL || c.ldY * (int64_t) es > 0x7fffffffLL) {
		set_error("%s: rows of Y and W are at most 2 GiB apart", what);
		return -CLA_ERR_UNSUPPORTED;
	}
	return 0;
}

static int forward(const GateCall& c, hipStream_t stream) {
	const char* what = "gate";
	int rc = check_operands(what, c);
	if(rc) return rc;
	const size_t es = type_bytes(c.type);
	if(c.m > 0 && (rc = check_operand(what, "the output", c.out, c.m, c.nOut, c.ldOut, es, es))) return rc;
	return (rc = check_ready()) ? rc : launch_gate(c, stream);
}

static int backward(const GateCall& c, int64_t wsBytes, hipStream_t stream) {
	const char* what = "gate_backward";
	int rc = check_operands(what, c);
	if(rc) return rc;
	const size_t es = type_bytes(c.type);
	if(!c.dY && !c.dW && !c.dB) { set_error("%s: no gradient is asked for", what); return -CLA_ERR_INVALID; }
	if(c.m > 0 && (rc = check_operand(what, "the incoming gradient", c.D, c.m, c.nOut, c.ldD, es, es))) return rc;
	if(c.dY && (rc = check_operand(what, "the gradient of Y", c.dY, c.m, c.nIn, c.ldDY, es, es))) return rc;
	if(c.dW && (rc = check_operand(what, "the gradient of W", c.dW, 2 * (int64_t) c.nOut, c.nIn, c.ldDW, es, es))) return rc;
	if(((uintptr_t) c.dB & (es - 1)) != 0) { set_error("%s: the gradient of the bias is not aligned", what); return -CLA_ERR_INVALID; }
	if((rc = check_ready())) return rc;
	const int64_t need = c.m > 0 ? (int64_t) gate_plan(c.type, c.m, c.nIn, c.nOut).bytes : 0;
	if(need > 0 && (!c.ws || ((uintptr_t) c.ws & 15) || wsBytes < need)) {
		set_error("%s: a workspace of %lld bytes, aligned to 16, is needed (%lld given)", what, (long long) need, c.ws ? (long long) wsBytes : 0LL);
		return -CLA_ERR_INVALID;
	}
	return launch_gate_backward(c, stream);
}

static GateCall call_of(int act, int type, const void* Y, int64_t m, int nIn, int64_t ldY, const void* W, int64_t ldW, const void* bias, int nOut) {
	GateCall c{};
	c.act = act; c.type = type;
	c.Y = Y; c.m = m; c.nIn = nIn; c.ldY = ldY;
	c.W = W; c.ldW = ldW; c.bias = bias; c.nOut = nOut;
	return c;
}

// Device memory of a host form: freed behind its last wait, however the call ends.
struct GateStage {
	char* p = nullptr;
	size_t at = 0;
	~GateStage() { if(p) { (void) hipStreamSynchronize(nullptr); (void) hipFree(p); } }
	double* take(size_t doubles) { double* x = (double*) (p + at); at += up(doubles * 8, 256); return x; }
};

} // namespace cla

using namespace cla;

extern "C" {

int64_t cla_gate_workspace(int32_t type, int64_t nRowY, int32_t nIn, int32_t nOut, int32_t backward) {
	CLA_TRY
	const int rc = check_sizes("gate_workspace", type, nRowY, nIn, nOut);
	if(rc) return rc;
	return backward && nRowY > 0 ? (int64_t) gate_plan(type, nRowY, nIn, nOut).bytes : 0;
	CLA_CATCH_CODE(int64_t)
}

int cla_gate_dev_async(int32_t act, int32_t type, const void* dY, int64_t nRowY, int32_t nIn, int64_t ldY, const void* dW, int64_t ldW, const void* dBias, int32_t nOut,
	void* dOut, int64_t ldOut, void* dWorkspace, int64_t workspaceBytes, void* hipStream) {
	CLA_TRY
	(void) dWorkspace; (void) workspaceBytes;
	GateCall c = call_of(act, type, dY, nRowY, nIn, ldY, dW, ldW, dBias, nOut);
	c.out = dOut; c.ldOut = ldOut;
	return forward(c, (hipStream_t) hipStream);
	CLA_CATCH_CODE(int)
}

int cla_gate_backward_dev_async(int32_t act, int32_t type, const void* dY, int64_t nRowY, int32_t nIn, int64_t ldY, const void* dW, int64_t ldW, const void* dBias,
	int32_t nOut, const void* dGrad, int64_t ldGrad, void* dGradY, int64_t ldGradY, void* dGradW, int64_t ldGradW, void* dGradBias, void* dWorkspace,
	int64_t workspaceBytes, void* hipStream) {
	CLA_TRY
	GateCall c = call_of(act, type, dY, nRowY, nIn, ldY, dW, ldW, dBias, nOut);
	c.D = dGrad; c.ldD = ldGrad;
	c.dY = dGradY; c.ldDY = ldGradY;
	c.dW = dGradW; c.ldDW = ldGradW;
	c.dB = dGradBias;
	c.ws = (char*) dWorkspace;
	return backward(c, workspaceBytes, (hipStream_t) hipStream);
	CLA_CATCH_CODE(int)
}

int64_t cla_gate(int32_t act, const double* Y, int64_t nRowY, int32_t nIn, const double* W, const double* bias, int32_t nOut, double* out) {
	CLA_TRY
	GateCall c = call_of(act, CLA_F64, Y, nRowY, nIn, nIn, W, nIn, bias, nOut);
	c.out = out; c.ldOut = nOut;
	int rc = check_operands("gate", c);
	if(rc) return rc;
	if(nRowY > 0 && !out) { set_error("gate: the output is null"); return -CLA_ERR_INVALID; }
	if((rc = check_ready())) return rc;
	if(nRowY == 0) return 0;
	const size_t nY = (size_t) nRowY * nIn, nW = 2 * (size_t) nOut * nIn, nB = bias ? 2 * (size_t) nOut : 0, nO = (size_t) nRowY * nOut;
	GateStage s;
	if((rc = device_room("gate", (void**) &s.p, (nY + nW + nB + nO + 1) * 8 + 5 * 256))) return rc;
	double* const y = s.take(nY);
	double* const w = s.take(nW);
	double* const b = s.take(nB);
	double* const o = s.take(nO);
	CLA_HIP(hipMemcpyAsync(y, Y, nY * 8, hipMemcpyHostToDevice, nullptr));
	CLA_HIP(hipMemcpyAsync(w, W, nW * 8, hipMemcpyHostToDevice, nullptr));
	if(bias) CLA_HIP(hipMemcpyAsync(b, bias, nB * 8, hipMemcpyHostToDevice, nullptr));
	c.Y = y; c.W = w; c.bias = bias ? b : nullptr; c.out = o;
	if((rc = forward(c, nullptr))) return rc;
	CLA_HIP(hipMemcpyAsync(out, o, nO * 8, hipMemcpyDeviceToHost, nullptr));
	return count_nonzero(o, (int64_t) nO, (unsigned long long*) s.take(1), nullptr);
	CLA_CATCH_CODE(int64_t)
}

int cla_gate_backward(int32_t act, const double* Y, int64_t nRowY, int32_t nIn, const double* W, const double* bias, int32_t nOut, const double* grad, double* gradY,
	double* gradW, double* gradBias) {
	CLA_TRY
	GateCall c = call_of(act, CLA_F64, Y, nRowY, nIn, nIn, W, nIn, bias, nOut);
	int rc = check_operands("gate_backward", c);
	if(rc) return rc;
	if((nRowY > 0 && !grad) || (!gradY && !gradW && !gradBias)) { set_error("gate_backward: %s", grad ? "no gradient is asked for" : "the incoming gradient is null"); return -CLA_ERR_INVALID; }
	if((rc = check_ready())) return rc;
	const size_t nY = (size_t) nRowY * nIn, nW = 2 * (size_t) nOut * nIn, nB = 2 * (size_t) nOut, nO = (size_t) nRowY * nOut;
	const int64_t wsBytes = cla_gate_workspace(CLA_F64, nRowY, nIn, nOut, 1);
	GateStage s;
	if((rc = device_room("gate_backward", (void**) &s.p, (2 * nY + 2 * nW + 2 * nB + nO) * 8 + 8 * 256 + (size_t) wsBytes))) return rc;
	double* const y = s.take(nY);
	double* const w = s.take(nW);
	double* const b = s.take(nB);
	double* const d = s.take(nO);
	double* const gy = s.take(nY);
	double* const gw = s.take(nW);
	double* const gb = s.take(nB);
	if(nRowY > 0) {
		CLA_HIP(hipMemcpyAsync(y, Y, nY * 8, hipMemcpyHostToDevice, nullptr));
		CLA_HIP(hipMemcpyAsync(d, grad, nO * 8, hipMemcpyHostToDevice, nullptr));
	}
	CLA_HIP(hipMemcpyAsync(w, W, nW * 8, hipMemcpyHostToDevice, nullptr));
	if(bias) CLA_HIP(hipMemcpyAsync(b, bias, nB * 8, hipMemcpyHostToDevice, nullptr));
	c.Y = y; c.W = w; c.bias = bias ? b : nullptr;
	c.D = d; c.ldD = nOut;
	if(gradY && nRowY > 0) { c.dY = gy; c.ldDY = nIn; }
	if(gradW) { c.dW = gw; c.ldDW = nIn; }
	if(gradBias) c.dB = gb;
	c.ws = s.p + s.at;
	if((c.dY || c.dW || c.dB) && (rc = backward(c, wsBytes, nullptr))) return rc;
	if(c.dY) CLA_HIP(hipMemcpyAsync(gradY, gy, nY * 8, hipMemcpyDeviceToHost, nullptr));
	if(gradW) CLA_HIP(hipMemcpyAsync(gradW, gw, nW * 8, hipMemcpyDeviceToHost, nullptr));
	if(gradBias) CLA_HIP(hipMemcpyAsync(gradBias, gb, nB * 8, hipMemcpyDeviceToHost, nullptr));
	CLA_HIP(hipStreamSynchronize(nullptr));
	return 0;
	CLA_CATCH_CODE(int)
}

} // extern "C"
