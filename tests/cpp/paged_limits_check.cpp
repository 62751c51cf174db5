// What the paged cache's calls find out about their arguments (csrc/paged_plan.h), for a test on the CPU.
#include "paged_plan.h"

using namespace nvfp4::paged;

extern "C" {

// Whether a sequence's rows or positions are cut off; -1: the batch is refused.
int paged_cut_off(const nvfp4_kv_cache* c, const nvfp4_paged_batch* b, int s) {
    Batch x{};
    return check_batch(c, b, &x) ? -1 : cut_off(x, s);
}

unsigned int limits_reported(unsigned int wait, unsigned int place) { return reported(wait, place); }
int limits_check_append(const nvfp4_kv_append_desc* d) {
    AppendArgs a{};
    bool empty = false;
    return check_append(d, &a, &empty);
}
int limits_check_attention(const nvfp4_paged_attention_desc* d) {
    AttentionArgs a{};
    bool empty = false;
    return check_attention(d, &a, &empty);
}

}  // extern "C"
