// Gated units of __bf16 (k_gate_impl.hpp).
#include "k_gate_impl.hpp"

namespace cla {

template int gate_forward<__bf16>(const GateCall& c, hipStream_t stream);
template int gate_backward<__bf16>(const GateCall& c, hipStream_t stream);

} // namespace cla
