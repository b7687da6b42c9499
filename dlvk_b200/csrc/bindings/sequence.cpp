// Bindings of the operators over sequences with a state and of the choice of
// the next word.
#include "bind_common.h"

namespace dlvk {
namespace bind {

using namespace ::dlvk::aten;

void register_sequence(py::module& m) {
  m.def("short_conv_fwd", &short_conv_fwd_op, py::arg("x"), py::arg("weight"), py::arg("bias") = py::none(),
        py::arg("state") = py::none(), py::arg("lengths") = py::none(), py::arg("silu") = true,
        py::arg("want_state") = false, py::arg("out_state") = py::none());
  m.def("short_conv_step", &short_conv_step_op, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("state"),
        py::arg("silu") = true, py::arg("out_state") = py::none());
  m.def("state_scan_step", &state_scan_step_op, py::arg("u"), py::arg("dt"), py::arg("a_log"), py::arg("b"),
        py::arg("c"), py::arg("state"), py::arg("skip") = py::none(), py::arg("z") = py::none(),
        py::arg("dt_bias") = py::none(), py::arg("out_state") = py::none());
  m.def("short_conv_bwd", &short_conv_bwd_op, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("dy"),
        py::arg("state") = py::none(), py::arg("lengths") = py::none(), py::arg("silu") = true,
        py::arg("dx") = py::none(), py::arg("dweight") = py::none(), py::arg("dbias") = py::none(),
        py::arg("accumulate") = false);
  m.def("state_scan_fwd", &state_scan_fwd_op, py::arg("u"), py::arg("dt"), py::arg("a_log"), py::arg("b"), py::arg("c"),
        py::arg("skip") = py::none(), py::arg("z") = py::none(), py::arg("dt_bias") = py::none(),
        py::arg("state") = py::none(), py::arg("lengths") = py::none(), py::arg("want_state") = false,
        py::arg("save") = false, py::arg("out_state") = py::none());
  m.def("state_scan_bwd", &state_scan_bwd_op, py::arg("u"), py::arg("dt"), py::arg("a_log"), py::arg("b"), py::arg("c"),
        py::arg("skip"), py::arg("z"), py::arg("dt_bias"), py::arg("dy"), py::arg("saved"),
        py::arg("lengths") = py::none(), py::arg("du") = py::none(), py::arg("ddt") = py::none(),
        py::arg("db") = py::none(), py::arg("dc") = py::none(), py::arg("dz") = py::none(),
        py::arg("da_log") = py::none(), py::arg("dskip") = py::none(), py::arg("ddt_bias") = py::none(),
        py::arg("accumulate") = false);
  m.def("sample_tokens", &sample_tokens_op, py::arg("logits"), py::arg("uniform"), py::arg("temperature") = 1.0,
        py::arg("top_k") = 0, py::arg("top_p") = 1.0, py::arg("min_p") = 0.0, py::arg("temperatures") = py::none(),
        py::arg("top_ks") = py::none(), py::arg("top_ps") = py::none(), py::arg("min_ps") = py::none());
}

}  // namespace bind
}  // namespace dlvk
