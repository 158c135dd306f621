// Attention over the 4-bit cache through a window beside a sequence's first tokens: the kernels of
// attention_kv4.hpp over two ranges of its keys, one after the other. Steps of the first tokens come first, the
// keys between them and the window are not read. One token of 64 sequences, 4 query heads to each of 8 cache
// heads, a window of 4,096 and 64 first tokens: 291 MB in 51 us, 5.6 TB/s; a prompt of 8,192 tokens through 2,000
// keys and 100 first ones 335 us, 0.73 PFLOP/s, bound as attention_kv4's prompts are and idle for 11 % of the time
// behind the last, shorter tiles (along one line of keys 480).
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
