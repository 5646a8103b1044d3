// What the entry points of 8-bit matrices and gated units share (cla_q8.hip holds the code).
#pragma once
#include "cla_internal.hpp"

namespace cla {

inline size_t up(size_t x, size_t to) { return (x + to - 1) / to * to; }
size_t type_bytes(int type);
int check_type(const char* what, int type);
int check_act(const char* what, int act);
int check_rows(const char* what, int64_t m);
// A row-major operand: there, aligned to `to` bytes, rows that do not overlap, its bytes within 63 bits.
int check_operand(const char* what, const char* name, const void* p, int64_t rows, int64_t cols, int64_t ld, size_t es, size_t to);
// Device memory for a call; where there is none, the runtime's error does not stay for the next call to find.
int device_room(const char* what, void** p, size_t bytes);
// Rows that one launch of tiles of tm x tn on 256 threads takes of a product with so many columns (shapes with more threads have as much larger tiles).
inline int64_t rows_of_a_launch(int64_t tm, int64_t tn, int64_t cols) { return LAUNCH_THREADS / 256 / ((cols + tn - 1) / tn) * tm; }
// Non-zeros of n values on the device; waits for the stream.
int64_t count_nonzero(const double* x, int64_t n, unsigned long long* dCount, hipStream_t stream);

} // namespace cla
