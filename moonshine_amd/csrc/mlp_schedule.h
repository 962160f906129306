// Where a stage of the fused encoder MLP kernel (k_mlp.hip) waits for the stage behind it.  Plain C++: tests/c/mlp_schedule.cpp walks it.
#pragma once

namespace msh {

// A stage of `nf` steps reads its operand fragments `pf` steps ahead, so its steps nf - pf and later read the NEXT stage's.  Behind step
// mlp_publish_step() the workgroup waits for the next stage's bytes and passes the barrier that publishes them; a step's read follows the
// barrier of the same step.  The middle of the stage, unless the next stage's fragments are read before it: a first stage of four steps
// (hidden size 64) reads them from its step 0 on.
constexpr int mlp_publish_step(int nf, int pf, bool last) { return last || nf - pf >= nf / 2 ? nf / 2 : nf - pf; }

}  // namespace msh
