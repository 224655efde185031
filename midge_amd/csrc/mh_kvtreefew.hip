// mh_kvtreefew.hip — mh_kv_tree_attention_dev where a sequence has few columns.
#include "mh_kvfew.cuh"

namespace mh {

int kv_few_tree_run(const mh_kv_cache &c, const mh_kv_batch &b, KvAttnArgs A, void *ws) { return few_run<true>(c, b, A, ws); }

}  // namespace mh
