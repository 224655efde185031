// mh_kvtreemany.hip — mh_kv_tree_attention_dev where a sequence has many columns.
#include "mh_kvmany.cuh"

namespace mh {

int kv_many_tree_run(const mh_kv_cache &c, const mh_kv_batch &b, KvAttnArgs A, void *ws) { return many_run<true>(c, b, A, ws); }

}  // namespace mh
