// A context without a device, whose buffers are made-up addresses: for calls that the library refuses before it touches the GPU.
#include "../p0pc0rn_b200/csrc/internal.h"

extern "C" p0_ctx *host_ctx() { return new p0_ctx(); }
extern "C" void host_buf(p0_ctx *c, uint64_t id, uint64_t address, uint64_t bytes) {
  P0Buffer b;
  b.ptr = (void *)(uintptr_t)address;
  b.bytes = bytes;
  b.owned = false;
  c->bufs[id] = b;
}
extern "C" void host_free(p0_ctx *c) { delete c; }
