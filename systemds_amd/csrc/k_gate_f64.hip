// Gated units of double (k_gate_impl.hpp).
#include "k_gate_impl.hpp"

namespace cla {

template int gate_forward<double>(const GateCall& c, hipStream_t stream);
template int gate_backward<double>(const GateCall& c, hipStream_t stream);

} // namespace cla
