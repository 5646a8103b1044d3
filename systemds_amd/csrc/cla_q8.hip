// Entry points of the 8-bit matrices (include/cla_hip.h): handles, checks of arguments, host forms. The kernels are in k_q8.hip.
#include "../../include/cla_hip.h"
#include "k_q8.hpp"
#include "cla_layers.hpp"
#include <algorithm>
#include <cstring>

struct cla_q8 {
	int64_t nRows = 0, ldW = 0;
	int32_t nCols = 0;
	bool set = false;
	int8_t* dW = nullptr;     // nCols rows of ldW bytes (a multiple of 128, zeros behind nRows)
	float* dScale = nullptr;
	hipStream_t stream = nullptr;
	bool ownStream = false;
	std::recursive_mutex mu;
	void* dStage = nullptr;   // operands and result of the host forms
	size_t stageCap = 0;
};

namespace cla {

int check_type(const char* what, int type) {
	if(type >= CLA_F64 && type <= CLA_F16) return 0;
	set_error("%s: unknown element type %d", what, type);
	return -CLA_ERR_INVALID;
}
size_t type_bytes(int type) { return type == CLA_F64 ? 8 : type == CLA_F32 ? 4 : 2; }

int check_act(const char* what, int act) {
	if(act >= CLA_ACT_SIGMOID && act <= CLA_ACT_NONE) return 0;
	set_error("%s: unknown activation %d", what, act);
	return -CLA_ERR_INVALID;
}

int check_operand(const char* what, const char* name, const void* p, int64_t rows, int64_t cols, int64_t ld, size_t es, size_t to) {
	if(!p || ((uintptr_t) p & (to - 1)) != 0) { set_error("%s: %s is %s", what, name, p ? "not aligned" : "null"); return -CLA_ERR_INVALID; }
	if(ld < cols || ld > ((int64_t) 1 << 40) || rows > 0x7fffffffLL || ld * (double) es * (double) std::max<int64_t>(rows, 1) > 9e18) {
		set_error("%s: leading dimension %lld of %s (%lld x %lld)", what, (long long) ld, name, (long long) rows, (long long) cols);
		return -CLA_ERR_INVALID;
	}
	return 0;
}

int check_rows(const char* what, int64_t m) {
	if(m >= 0 && m <= 0x7fffffffLL) return 0;
	set_error("%s: %lld rows", what, (long long) m);
	return -CLA_ERR_INVALID;
}

int device_room(const char* what, void** p, size_t bytes) {
	if(!no_room(p, bytes)) return 0;
	set_error("%s: %zu bytes of device memory could not be allocated", what, bytes);
	return -CLA_ERR_DEVICE;
}

__global__ __launch_bounds__(256) void k_count_nonzero(const double* __restrict__ x, int64_t n, unsigned long long* __restrict__ count) {
	unsigned long long c = 0;
	for(int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t) gridDim.x * 256) c += x[i] != 0.0;
#pragma unroll
	for(int d = 32; d > 0; d >>= 1) c += __shfl_xor(c, d, 64);
	if((threadIdx.x & 63) == 0 && c != 0) atomicAdd(count, c);
}

int64_t count_nonzero(const double* x, int64_t n, unsigned long long* dCount, hipStream_t stream) {
	unsigned long long c = 0;
	CLA_HIP(hipMemsetAsync(dCount, 0, sizeof(c), stream));
	if(n > 0) k_count_nonzero<<<(unsigned) std::min<int64_t>((n + 255) / 256, g_numCU * 8), 256, 0, stream>>>(x, n, dCount);
	CLA_HIP(hipGetLastError());
	CLA_HIP(hipMemcpyAsync(&c, dCount, sizeof(c), hipMemcpyDeviceToHost, stream));
	CLA_HIP(hipStreamSynchronize(stream));
	return (int64_t) c;
}

static int64_t ld_rows(const cla_q8* h) { return (int64_t) up((size_t) h->nRows, 16); }

static int check_q8(cla_q8* h, bool set) {
	if(!h) { set_error("null 8-bit matrix handle"); return -CLA_ERR_INVALID; }
	if(set && !h->set) { set_error("8-bit matrix without values"); return -CLA_ERR_STATE; }
	return check_ready();
}

// What is on its way on a stream that the handle was on before, or in a graph's replay, still reads the values that are about to be replaced.
static int wait_for_readers(cla_q8* h) {
	if(h->set) CLA_HIP(hipDeviceSynchronize());
	return 0;
}

struct DevTmp { // device memory of a call that waits
	void* p = nullptr;
	~DevTmp() { if(p) (void) hipFree(p); }
};

static int product(cla_q8* h, bool gated, int act, const int8_t* Q, int64_t ldQ, const float* s, int64_t m, const void* bias, void* out, int type,
	int64_t ldOut, const void* Y = nullptr, int64_t ldY = 0) {
	Q8Product p{};
	p.W = h->dW; p.ldW = h->ldW; p.t = h->dScale;
	p.Q = Q; p.ldQ = ldQ; p.s = s; p.m = m;
	p.K = (int32_t) h->nRows; p.N = h->nCols; p.act = act;
	p.bias = bias; p.out = out; p.ldOut = ldOut;
	p.Y = Y; p.ldY = ldY;
	const int64_t rows = rows_of_a_launch(64, 128, h->nCols); // (tiles of the smallest shape)
	for(int64_t r = 0; r < m; r += rows) {
		p.m = std::min(m - r, rows);
		if(Q) { p.Q = Q + r * ldQ; p.s = s + r; }
		p.out = (char*) out + r * ldOut * (int64_t) type_bytes(type);
		if(const int rc = launch_q8(p, type, gated, h->stream)) return rc;
	}
	return 0;
}

static int check_out(cla_q8* h, const char* what, bool gated, int act, int64_t m, const void* bias, const void* out, int type, int64_t ldOut) {
	int rc;
	if((rc = check_type(what, type)) || (rc = check_rows(what, m))) return rc;
	if(gated && (rc = check_act(what, act))) return rc;
	if(gated && (h->nCols & 1)) { set_error("%s: a gated unit has an even number of columns (%d)", what, h->nCols); return -CLA_ERR_INVALID; }
	const size_t es = type_bytes(type);
	if(((uintptr_t) bias & (es - 1)) != 0) { set_error("%s: bias is not aligned", what); return -CLA_ERR_INVALID; }
	return m == 0 ? 0 : check_operand(what, "the output", out, m, gated ? h->nCols / 2 : h->nCols, ldOut, es, es);
}

static int from_rows(cla_q8* h, const char* what, bool gated, int act, const void* dY, int type, int64_t m, int64_t ldY, const void* dBias, void* dOut, int64_t ldOut,
	void* ws, int64_t wsBytes) {
	int rc = check_q8(h, true);
	if(rc || (rc = check_out(h, what, gated, act, m, dBias, dOut, type, ldOut))) return rc;
	if(m == 0) return 0;
	const size_t es = type_bytes(type);
	if((rc = check_operand(what, "Y", dY, m, h->nRows, ldY, es, es))) return rc;
	const int64_t need = cla_q8_workspace(h, m);
	if(!ws || ((uintptr_t) ws & 15) || wsBytes < need) {
		set_error("%s: a workspace of %lld bytes, aligned to 16, is needed (%lld given)", what, (long long) need, ws ? (long long) wsBytes : 0LL);
		return -CLA_ERR_INVALID;
	}
	std::lock_guard<std::recursive_mutex> lk(h->mu);
	if(q8_fuses(m, h->nRows)) return product(h, gated, act, nullptr, 0, nullptr, m, dBias, dOut, type, ldOut, dY, ldY);
	float* const s = (float*) ws;
	int8_t* const q = (int8_t*) ws + up((size_t) m * sizeof(float), 256);
	const int64_t ldQ = ld_rows(h);
	if((rc = launch_q8_rows(dY, type, m, (int) h->nRows, ldY, q, ldQ, s, h->stream))) return rc;
	return product(h, gated, act, q, ldQ, s, m, dBias, dOut, type, ldOut);
}

static int from_quantized(cla_q8* h, const char* what, bool gated, int act, const int8_t* dQ, int64_t ldQ, const float* dScale, int64_t m, const void* dBias, void* dOut,
	int type, int64_t ldOut) {
	int rc = check_q8(h, true);
	if(rc || (rc = check_out(h, what, gated, act, m, dBias, dOut, type, ldOut))) return rc;
	if(m == 0) return 0;
	if((rc = check_operand(what, "the 8-bit rows", dQ, m, h->nRows, ldQ, 1, 16)) || (rc = check_operand(what, "the rows' scales", dScale, m, 1, 1, 4, 4))) return rc;
	if(ldQ & 15 || ldQ > ((int64_t) 4 << 20)) { set_error("%s: 8-bit rows are a multiple of 16 bytes apart, at most 4 MiB (%lld)", what, (long long) ldQ); return -CLA_ERR_INVALID; }
	std::lock_guard<std::recursive_mutex> lk(h->mu);
	return product(h, gated, act, dQ, ldQ, dScale, m, dBias, dOut, type, ldOut);
}

// The host forms: operands and result staged on the device, the workspace behind them.
static int64_t host_product(cla_q8* h, const char* what, bool gated, int act, const double* Y, int64_t m, const double* bias, double* out) {
	int rc = check_q8(h, true);
	if(rc) return rc;
	if((rc = check_out(h, what, gated, act, m, bias, out, CLA_F64, h->nCols))) return rc;
	if(m == 0) return 0;
	if(!Y) { set_error("%s: Y is null", what); return -CLA_ERR_INVALID; }
	const int64_t n = gated ? h->nCols / 2 : h->nCols;
	std::lock_guard<std::recursive_mutex> lk(h->mu);
	const size_t bY = up((size_t) m * h->nRows * 8, 256), bB = up(bias ? (size_t) h->nCols * 8 : 0, 256), bO = up((size_t) m * n * 8, 256);
	const size_t bW = up((size_t) cla_q8_workspace(h, m), 256), need = bY + bB + bO + bW + 256;
	if(need > h->stageCap) {
		if(h->dStage) CLA_HIP(hipFree(h->dStage)); // (no call of a host form is under way)
		h->dStage = nullptr; h->stageCap = 0;
		if(int r = device_room(what, &h->dStage, need)) return r;
		h->stageCap = need;
	}
	char* const base = (char*) h->dStage;
	double* const dB = (double*) (base + bY);
	double* const dO = (double*) (base + bY + bB);
	CLA_HIP(hipMemcpyAsync(base, Y, (size_t) m * h->nRows * 8, hipMemcpyHostToDevice, h->stream));
	if(bias) CLA_HIP(hipMemcpyAsync(dB, bias, (size_t) h->nCols * 8, hipMemcpyHostToDevice, h->stream));
	if((rc = from_rows(h, what, gated, act, base, CLA_F64, m, h->nRows, bias ? dB : nullptr, dO, n, base + bY + bB + bO, (int64_t) bW))) return rc;
	CLA_HIP(hipMemcpyAsync(out, dO, (size_t) m * n * 8, hipMemcpyDeviceToHost, h->stream));
	return count_nonzero(dO, m * n, (unsigned long long*) (base + bY + bB + bO + bW), h->stream);
}

} // namespace cla

using namespace cla;

extern "C" {

int cla_quantize_rows_dev_async(const void* dY, int32_t type, int64_t nRowY, int32_t k, int64_t ldY, int8_t* dQ, int64_t ldQ, float* dScale, void* hipStream) {
	CLA_TRY
	const char* what = "quantize_rows";
	int rc;
	if((rc = check_type(what, type)) || (rc = check_rows(what, nRowY))) return rc;
	if(k <= 0 || k > 1 << 30) { set_error("%s: rows of %d values", what, k); return -CLA_ERR_INVALID; } // (beyond 2^30 places in a row leave 32 bits)
	if(nRowY == 0) return check_ready();
	const size_t es = type_bytes(type);
	if((rc = check_operand(what, "Y", dY, nRowY, k, ldY, es, es)) || (rc = check_operand(what, "the 8-bit rows", dQ, nRowY, k, ldQ, 1, 1)) ||
		(rc = check_operand(what, "the scales", dScale, nRowY, 1, 1, 4, 4)) || (rc = check_ready()))
		return rc;
	return launch_q8_rows(dY, type, nRowY, k, ldY, dQ, ldQ, dScale, (hipStream_t) hipStream);
	CLA_CATCH_CODE(int)
}

int cla_block_quantize_rows_dev_async(cla_handle b, int8_t* dQ, int64_t ldQ, float* dScale) {
	CLA_TRY
	const char* what = "block_quantize_rows";
	if(!b) { set_error("null block handle"); return -CLA_ERR_INVALID; }
	if(!b->finalized) { set_error("block not finalized"); return -CLA_ERR_STATE; }
	int rc = check_ready();
	if(rc) return rc;
	if(b->nRows == 0) return 0;
	if((rc = check_operand(what, "the 8-bit rows", dQ, b->nRows, b->nCols, ldQ, 1, 1)) || (rc = check_operand(what, "the scales", dScale, b->nRows, 1, 1, 4, 4))) return rc;
	std::lock_guard<std::recursive_mutex> lk(b->mu);
	clear_stats(b);
	const int64_t bytes = (int64_t) b->nCols * 8, chunk = std::min<int64_t>(b->nRows, std::max<int64_t>(1, ((int64_t) 64 << 20) / bytes));
	// One chunk for the block's calls, each of which waits for the last use of it on the device (the block may have changed streams); one of its own for a call that is being
	// captured, since its graph may be replayed beside any other.
	hipStreamCaptureStatus capturing = hipStreamCaptureStatusNone;
	CLA_HIP(hipStreamIsCapturing(b->stream, &capturing));
	double* rows = b->dQuantRows;
	if(capturing != hipStreamCaptureStatusNone) {
		b->wsOld.reserve(b->wsOld.size() + 1);
		hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed; // (an allocation is none of the stream's work)
		CLA_HIP(hipThreadExchangeStreamCaptureMode(&mode));
		rc = device_room(what, (void**) &rows, (size_t) (chunk * bytes));
		CLA_HIP(hipThreadExchangeStreamCaptureMode(&mode));
		if(rc) return rc;
		b->wsOld.push_back(rows);
	}
	else {
		if(!rows && (rc = device_room(what, (void**) &rows, (size_t) (chunk * bytes)))) return rc;
		b->dQuantRows = rows;
		if(b->quantDone) CLA_HIP(hipStreamWaitEvent(b->stream, b->quantDone, 0));
		else CLA_HIP(hipEventCreateWithFlags(&b->quantDone, hipEventDisableTiming));
	}
	for(int64_t r0 = 0; r0 < b->nRows && !rc; r0 += chunk) {
		const int64_t r1 = std::min(b->nRows, r0 + chunk);
		if((rc = launch_decompress_rows(b, r0, r1, rows))) break;
		Prof pf(b, "k_q8_rows", (long) (r1 - r0), 256, 0, (double) (r1 - r0) * (bytes + b->nCols + 4));
		rc = launch_q8_rows(rows, CLA_F64, r1 - r0, b->nCols, b->nCols, dQ + r0 * ldQ, ldQ, dScale + r0, b->stream);
	}
	if(capturing == hipStreamCaptureStatusNone) CLA_HIP(hipEventRecord(b->quantDone, b->stream));
	return rc;
	CLA_CATCH_CODE(int)
}

cla_q8_handle cla_q8_create(int64_t nRows, int32_t nCols) {
	CLA_TRY
	if(check_ready()) return nullptr;
	if(nRows <= 0 || nCols <= 0 || nRows > Q8_MAX_K || nCols > Q8_MAX_N) {
		set_error("invalid 8-bit matrix %lld x %d (at most %d x %d)", (long long) nRows, nCols, Q8_MAX_K, Q8_MAX_N);
		return nullptr;
	}
	cla_q8* h = new cla_q8();
	h->nRows = nRows; h->nCols = nCols;
	h->ldW = (int64_t) up((size_t) nRows, 128);
	if(hipStreamCreate(&h->stream) != hipSuccess) { set_error("hipStreamCreate failed"); delete h; return nullptr; }
	h->ownStream = true;
	if(hipMalloc((void**) &h->dW, (size_t) h->ldW * nCols) != hipSuccess || hipMalloc((void**) &h->dScale, sizeof(float) * (size_t) nCols) != hipSuccess ||
		hipMemset(h->dW, 0, (size_t) h->ldW * nCols) != hipSuccess || hipStreamSynchronize(nullptr) != hipSuccess) {
		(void) hipGetLastError();
		set_error("an 8-bit matrix of %lld x %d could not be allocated", (long long) nRows, nCols);
		cla_q8_free(h);
		return nullptr;
	}
	return h;
	CLA_CATCH_NULL
}

void cla_q8_free(cla_q8_handle h) {
	CLA_TRY
	if(!h) return;
	(void) check_ready();
	(void) hipStreamSynchronize(h->stream);
	if(h->dW) (void) hipFree(h->dW);
	if(h->dScale) (void) hipFree(h->dScale);
	if(h->dStage) (void) hipFree(h->dStage);
	if(h->ownStream && h->stream) (void) hipStreamDestroy(h->stream);
	delete h;
	CLA_CATCH_VOID
}

int cla_q8_set_stream(cla_q8_handle h, void* hipStream) {
	CLA_TRY
	int rc = check_q8(h, false);
	if(rc) return rc;
	std::lock_guard<std::recursive_mutex> lk(h->mu);
	if(h->ownStream && h->stream) { (void) hipStreamSynchronize(h->stream); (void) hipStreamDestroy(h->stream); }
	h->stream = (hipStream_t) hipStream;
	h->ownStream = false;
	return 0;
	CLA_CATCH_CODE(int)
}

int cla_q8_set_dev(cla_q8_handle h, const void* dW, int32_t type, int64_t ld, int32_t byColumn) {
	CLA_TRY
	const char* what = "q8_set";
	int rc = check_q8(h, false);
	if(rc || (rc = check_type(what, type))) return rc;
	const size_t es = type_bytes(type);
	if((rc = check_operand(what, "W", dW, byColumn ? h->nCols : h->nRows, byColumn ? h->nRows : h->nCols, ld, es, es))) return rc;
	std::lock_guard<std::recursive_mutex> lk(h->mu);
	DevTmp tmp;
	if((rc = wait_for_readers(h))) return rc;
	if(byColumn) rc = launch_q8_rows(dW, type, h->nCols, (int) h->nRows, ld, h->dW, h->ldW, h->dScale, h->stream);
	else {
		if((rc = device_room(what, &tmp.p, (size_t) h->nRows * h->nCols * 8))) return rc;
		rc = launch_q8_columns(dW, type, ld, h->nRows, h->nCols, (double*) tmp.p, h->stream);
		if(!rc) rc = launch_q8_rows(tmp.p, CLA_F64, h->nCols, (int) h->nRows, h->nRows, h->dW, h->ldW, h->dScale, h->stream);
	}
	const hipError_t e = hipStreamSynchronize(h->stream);
	if(rc) return rc;
	CLA_HIP(e);
	h->set = true;
	return 0;
	CLA_CATCH_CODE(int)
}

int cla_q8_set(cla_q8_handle h, const double* W) {
	CLA_TRY
	int rc = check_q8(h, false);
	if(rc) return rc;
	if(!W) { set_error("q8_set: W is null"); return -CLA_ERR_INVALID; }
	std::lock_guard<std::recursive_mutex> lk(h->mu);
	DevTmp tmp;
	const size_t bytes = (size_t) h->nRows * h->nCols * 8;
	if((rc = device_room("q8_set", &tmp.p, bytes))) return rc;
	CLA_HIP(hipMemcpyAsync(tmp.p, W, bytes, hipMemcpyHostToDevice, h->stream));
	rc = cla_q8_set_dev(h, tmp.p, CLA_F64, h->nCols, 0);
	(void) hipStreamSynchronize(h->stream);
	return rc;
	CLA_CATCH_CODE(int)
}

int cla_q8_set_values_dev(cla_q8_handle h, const int8_t* dValues, int64_t ld, int32_t byColumn, const float* dScales) {
	CLA_TRY
	const char* what = "q8_set_values";
	int rc = check_q8(h, false);
	if(rc || (rc = check_operand(what, "the values", dValues, byColumn ? h->nCols : h->nRows, byColumn ? h->nRows : h->nCols, ld, 1, 1)) ||
		(rc = check_operand(what, "the scales", dScales, 1, h->nCols, h->nCols, 4, 4)))
		return rc;
	std::lock_guard<std::recursive_mutex> lk(h->mu);
	if((rc = wait_for_readers(h)) || (rc = launch_q8_layout(dValues, ld, byColumn, h->nRows, h->nCols, h->dW, h->ldW, h->stream))) return rc;
	CLA_HIP(hipMemcpyAsync(h->dScale, dScales, sizeof(float) * (size_t) h->nCols, hipMemcpyDeviceToDevice, h->stream));
	CLA_HIP(hipStreamSynchronize(h->stream));
	h->set = true;
	return 0;
	CLA_CATCH_CODE(int)
}

int cla_q8_set_values(cla_q8_handle h, const int8_t* values, const float* scales) {
	CLA_TRY
	int rc = check_q8(h, false);
	if(rc) return rc;
	if(!values || !scales) { set_error("q8_set_values: null values or scales"); return -CLA_ERR_INVALID; }
	std::lock_guard<std::recursive_mutex> lk(h->mu);
	DevTmp v, s;
	const size_t n = (size_t) h->nRows * h->nCols;
	if((rc = device_room("q8_set_values", &v.p, n)) || (rc = device_room("q8_set_values", &s.p, sizeof(float) * (size_t) h->nCols))) return rc;
	CLA_HIP(hipMemcpyAsync(v.p, values, n, hipMemcpyHostToDevice, h->stream));
	CLA_HIP(hipMemcpyAsync(s.p, scales, sizeof(float) * (size_t) h->nCols, hipMemcpyHostToDevice, h->stream));
	rc = cla_q8_set_values_dev(h, (const int8_t*) v.p, h->nCols, 0, (const float*) s.p);
	(void) hipStreamSynchronize(h->stream);
	return rc;
	CLA_CATCH_CODE(int)
}

int cla_q8_get(cla_q8_handle h, int8_t* values, float* scales) {
	CLA_TRY
	int rc = check_q8(h, true);
	if(rc) return rc;
	if(!values || !scales) { set_error("q8_get: null values or scales"); return -CLA_ERR_INVALID; }
	std::lock_guard<std::recursive_mutex> lk(h->mu);
	std::vector<int8_t> w((size_t) h->ldW * h->nCols);
	CLA_HIP(hipMemcpyAsync(w.data(), h->dW, w.size(), hipMemcpyDeviceToHost, h->stream));
	CLA_HIP(hipMemcpyAsync(scales, h->dScale, sizeof(float) * (size_t) h->nCols, hipMemcpyDeviceToHost, h->stream));
	CLA_HIP(hipStreamSynchronize(h->stream));
	for(int64_t k = 0; k < h->nRows; k++)
		for(int32_t j = 0; j < h->nCols; j++) values[k * h->nCols + j] = w[(size_t) j * h->ldW + k];
	return 0;
	CLA_CATCH_CODE(int)
}

int64_t cla_q8_num_rows(cla_q8_handle h) { return h ? h->nRows : -CLA_ERR_INVALID; }
int32_t cla_q8_num_cols(cla_q8_handle h) { return h ? h->nCols : -CLA_ERR_INVALID; }
int64_t cla_q8_device_bytes(cla_q8_handle h) { return h ? h->ldW * h->nCols + (int64_t) sizeof(float) * h->nCols : -CLA_ERR_INVALID; }

int64_t cla_q8_workspace(cla_q8_handle h, int64_t nRowY) {
	CLA_TRY
	if(!h) { set_error("null 8-bit matrix handle"); return -CLA_ERR_INVALID; }
	const int rc = check_rows("q8_workspace", nRowY);
	return rc ? rc : (int64_t) up((size_t) nRowY * sizeof(float), 256) + nRowY * ld_rows(h);
	CLA_CATCH_CODE(int64_t)
}

int cla_q8_lmm_dev_async(cla_q8_handle h, const void* dY, int32_t type, int64_t nRowY, int64_t ldY, const void* dBias, void* dOut, int64_t ldOut, void* dWorkspace,
	int64_t workspaceBytes) {
	CLA_TRY
	return from_rows(h, "q8_lmm", false, 0, dY, type, nRowY, ldY, dBias, dOut, ldOut, dWorkspace, workspaceBytes);
	CLA_CATCH_CODE(int)
}

int cla_q8_gate_dev_async(cla_q8_handle h, int32_t act, const void* dY, int32_t type, int64_t nRowY, int64_t ldY, const void* dBias, void* dOut, int64_t ldOut,
	void* dWorkspace, int64_t workspaceBytes) {
	CLA_TRY
	return from_rows(h, "q8_gate", true, act, dY, type, nRowY, ldY, dBias, dOut, ldOut, dWorkspace, workspaceBytes);
	CLA_CATCH_CODE(int)
}

int cla_q8_lmm_quantized_dev_async(cla_q8_handle h, const int8_t* dQ, int64_t ldQ, const float* dScale, int64_t nRowY, const void* dBias, void* dOut, int32_t type,
	int64_t ldOut) {
	CLA_TRY
	return from_quantized(h, "q8_lmm_quantized", false, 0, dQ, ldQ, dScale, nRowY, dBias, dOut, type, ldOut);
	CLA_CATCH_CODE(int)
}

int cla_q8_gate_quantized_dev_async(cla_q8_handle h, int32_t act, const int8_t* dQ, int64_t ldQ, const float* dScale, int64_t nRowY, const void* dBias, void* dOut,
	int32_t type, int64_t ldOut) {
	CLA_TRY
	return from_quantized(h, "q8_gate_quantized", true, act, dQ, ldQ, dScale, nRowY, dBias, dOut, type, ldOut);
	CLA_CATCH_CODE(int)
}

int64_t cla_q8_lmm(cla_q8_handle h, const double* Y, int64_t nRowY, const double* bias, double* out) {
	CLA_TRY
	return host_product(h, "q8_lmm", false, 0, Y, nRowY, bias, out);
	CLA_CATCH_CODE(int64_t)
}

int64_t cla_q8_gate(cla_q8_handle h, int32_t act, const double* Y, int64_t nRowY, const double* bias, double* out) {
	CLA_TRY
	return host_product(h, "q8_gate", true, act, Y, nRowY, bias, out);
	CLA_CATCH_CODE(int64_t)
}

} // extern "C"
