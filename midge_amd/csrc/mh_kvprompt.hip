// mh_kvprompt.hip — mh_kv_attention_dev where a sequence has many columns.
#include "mh_kvmany.cuh"

namespace mh {

uint64_t kv_many_ws(const mh_kv_cache &c, const mh_kv_batch &b, int group) { return layout(b, group, c.head_dim, c.n_kv_heads).bytes; }

int kv_many_run(const mh_kv_cache &c, const mh_kv_batch &b, KvAttnArgs A, void *ws) { return many_run<false>(c, b, A, ws); }

}  // namespace mh
