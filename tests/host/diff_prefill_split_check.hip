// prefill_split_check.h with the settings of the differential 16-bit kernel, at
// each tile size.
#include "diff_prefill.hip"

#include "prefill_split_check.h"

int main() {
  return SplitCheck<clv::SplitCfg<128>>().run(clv::Shape<128>::kPairs, 256, 10000) |
         SplitCheck<clv::SplitCfg<256>>().run(clv::Shape<256>::kPairs, 256, 10000);
}
