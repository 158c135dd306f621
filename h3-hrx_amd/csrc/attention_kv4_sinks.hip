// Attention over the 4-bit cache through a window beside a sequence's first tokens: the kernels of
// attention_kv4.hpp over two ranges of its keys, one after the other. Steps of the first tokens come first, the
// keys between them and the window are not read.
#include "attention_kv4.hpp"

namespace h3 {

hipError_t launch_attention_kv4_sinks(const h3_kv4_cfg& cfg, const h3_kv4_attention_cfg& acfg,
                                      uint32_t sinks, const Kv4Plan& plan, uint32_t batch, uint32_t q_rows,
                                      uint32_t max_q, const Kv4Bindings& x, hipStream_t stream) {
  Args a = make_args(cfg, acfg, batch, q_rows, max_q, x);
  a.sinks = sinks;
  return launch_keys<kSinks>(cfg, a, plan, stream);
}

}  // namespace h3
