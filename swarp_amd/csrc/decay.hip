#include "learn.hpp"
extern "C" {
uint64_t swarp_decay_work_bytes(const swarp_decay_t *) { return 0; }
int swarp_decay_fwd(const swarp_decay_t *, void *) { return learn::fail("to come"); }
int swarp_decay_bwd(const swarp_decay_t *, void *) { return learn::fail("to come"); }
int swarp_decay_step(const swarp_decay_t *, void *) { return learn::fail("to come"); }
}
