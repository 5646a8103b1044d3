// Gated units of float (k_gate_impl.hpp).
#include "k_gate_impl.hpp"

namespace cla {

template int gate_forward<float>(const GateCall& c, hipStream_t stream);
template int gate_backward<float>(const GateCall& c, hipStream_t stream);

} // namespace cla
