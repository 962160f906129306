// The fused encoder MLP kernel's ring of operand stages (csrc/k_mlp.hip) step by step on the host, by the kernel's own rule for where a stage
// waits (csrc/mlp_schedule.h): which stages' bytes are in shared memory and published when a step reads, and whose buffer a copy refills.
#include "mlp_schedule.h"

using namespace msh;

// Hidden size d, `oproj` stages of the output projection (0: none) in front of nc chunks and the last stage; pf fragments ahead.
// Returns 0, or 1 + the stage that read bytes that were not published, or -1 - the stage whose buffer was refilled while it was read.
extern "C" int mlp_schedule_walk(int d, int oproj, int nc, int pf) {
  const int ks = d / 16, stages = (oproj ? (d / 32 + 1) / 2 : 0) + nc + 1, first = stages - nc - 1;
  int published = 1, copied = 1;   // the prologue: stages 0 and 1 are there
  for (int st = 0; st < stages; ++st) {
    const bool last = st == stages - 1, short_stage = st == first || last;
    const int nf = short_stage && st >= first ? ks : 2 * ks, mid = mlp_publish_step(nf, pf, last);
    if (mid < 0 || mid >= nf) return 1 + st;
    for (int f = 0; f < nf; ++f) {
      if (f == mid) {
        published = copied;              // every wave has waited for its pieces and passed the barrier
      } else if (f == mid + 1) {
        copied = st + 2;                 // the stage behind the next, into the buffer of the one before this
        if (copied % 3 == st % 3 || copied % 3 == (st + 1) % 3) return -1 - st;
      }
      const int reads = f + pf < nf ? st : st + 1;
      if (!(last && reads > st) && reads > published) return 1 + st;
    }
    if (mid + 1 >= nf) copied = st + 2;
    if (!last && st + 1 > published) return 1 + st;   // the next chunk's bias
  }
  return 0;
}
