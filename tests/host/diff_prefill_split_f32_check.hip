// prefill_split_check.h with the settings of the differential fp32 kernel, at
// each tile size and number of workgroups per compute unit. Twice its rows per
// workgroup: the check's batches have up to 64 query heads per kv head, and the
// schedule sees whole query tiles only.
#include "diff_prefill_f32.hip"

#include "prefill_split_check.h"

int main() {
  constexpr int rows = 2 * clv::kPairs;
  return SplitCheck<clv::SplitCfg<64>>().run(rows, 768, 10000) |
         SplitCheck<clv::SplitCfg<128>>().run(rows, 768, 10000) |
         SplitCheck<clv::SplitCfg<256>>().run(rows, 512, 10000);
}
