// The harness of paged_host.cpp with a communicator that no NCCL stands behind, and what the library knows of a tensor's memory.
#include "paged_host.cpp"

extern "C" {

void host_comm(cg_ctx* c) {
  c->comm = (void*)1;
  c->comm_world = 2;
}
// memory of the library's own, with a rounded copy of it
void host_known(cg_tensor* t) {
  auto copy = std::make_shared<Buffer>();
  copy->core = t->buf->core;
  copy->owned = false;
  t->buf->bf16_copy = copy;
  t->buf->owned = true;
  new std::shared_ptr<Buffer>(t->buf);  // (never freed)
  t->has_scalar = true;
}
int host_knows(const cg_tensor* t) { return (t->buf->bf16_copy ? 1 : 0) | (t->literal() ? 2 : 0) | (t->buf->rewritten ? 4 : 0); }

}
