// Gated units of _Float16 (k_gate_impl.hpp).
#include "k_gate_impl.hpp"

namespace cla {

template int gate_forward<_Float16>(const GateCall& c, hipStream_t stream);
template int gate_backward<_Float16>(const GateCall& c, hipStream_t stream);

} // namespace cla
