// One token step of a synthetic served model, run by the operators and checked
// against 64-bit oracles on the host: the serving diagnostic.
#pragma once

#include <cstdint>
#include <string>
#include <vector>

namespace serving {

struct StepResult {
  double ms = 0;          // a step
  double gbps = 0;        // codes, cache and logits read in a step, over its time
  double product_gbps = 0, attention_gbps = 0, logprob_gbps = 0;
  int64_t checked = 0;    // values compared with the oracles
  int64_t failures = 0;   // values beyond their bounds, or that differ between two runs
  std::vector<std::string> messages;  // the first few
};

// Throws std::runtime_error where the runtime fails. `oracle_offset` is added
// to what the oracles expect (0 but in tests of the comparison itself).
StepResult run_step(int device, int iters, uint32_t seed, double oracle_offset);

}  // namespace serving
