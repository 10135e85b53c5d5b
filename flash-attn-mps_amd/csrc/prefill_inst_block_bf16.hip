// BF16T prefill kernel variants over block-scaled E4M3 caches.
#include "prefill_kernel.h"

namespace fa_prefill {

PrefillChoiceOf<fa_block_attn> pick_block_bf16(int64_t d, bool causal, bool cap, bool win, int mk, bool split) {
  return pick_block<BF16T>(d, causal, cap, win, mk, split);
}

}  // namespace fa_prefill
