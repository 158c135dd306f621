// Attention over the 4-bit cache behind a prefix that all sequences share: the kernels of attention_kv4.hpp over
// the prefix's keys and then the sequence's own.
#include "attention_kv4.hpp"

namespace h3 {

hipError_t launch_attention_kv4_prefix(const h3_kv4_cfg& cfg, const h3_kv4_attention_cfg& acfg,
                                       uint32_t prefix_stride, const Kv4Plan& plan, uint32_t batch,
                                       uint32_t q_rows, uint32_t max_q, const Kv4Bindings& x,
                                       hipStream_t stream) {
  Args a = make_args(cfg, acfg, batch, q_rows, max_q, x);
  a.prefix_stride = prefix_stride;
  return launch_keys<kPrefix>(cfg, a, plan, stream);
}

}  // namespace h3
