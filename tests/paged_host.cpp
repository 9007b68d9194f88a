// Tensors and a context without a device, for the checks that the entry points make before they launch anything, and the index
// arithmetic of the kernels, compiled for the host out of their own header.
#include "paged.h"

using namespace cg;

extern "C" {

cg_ctx* host_ctx() {
  auto* c = new cg_ctx();       // (never freed: its destructor would call the device)
  auto* core = new std::shared_ptr<Core>(std::make_shared<Core>());
  c->core = *core;
  return c;
}
cg_tensor* host_tensor(cg_ctx* c, uint64_t address, int storage, int rank, const int64_t* dims, const int64_t* strides) {
  auto buf = std::make_shared<Buffer>();
  buf->core = c->core;
  buf->ptr = (void*)address;
  buf->owned = false;
  auto* t = new cg_tensor();
  t->ctx = c;
  t->tag = storage == ST_U32 ? CG_U32 : CG_F32;
  t->storage = storage;
  t->rank = rank;
  for (int i = 0; i < rank; ++i) { t->dims[i] = dims[i]; t->strides[i] = strides[i]; }
  t->buf = buf;
  return t;
}
void host_device(cg_tensor* t, int device) {
  auto core = std::make_shared<Core>();
  core->device = device;
  new std::shared_ptr<Core>(core);
  t->buf->core = core;
}

// (1: a row to be worked on) and its first token, count and length; *err as the kernels would leave it
int host_row_span(const uint32_t* starts, const uint32_t* lens, int64_t rows, int64_t cols, int lg, int64_t M, int64_t row, int64_t most, int64_t* out,
                  int32_t* err) {
  PagedRows p = {starts, lens, nullptr, rows, cols, M, 0, lg, err};
  return row_span(p, row, most, out, out + 1, out + 2);
}
int64_t host_page_of(const uint32_t* table, int64_t cols, int64_t n_pages, int lg, int64_t row, int64_t pos, int32_t* err) {
  PagedRows p = {nullptr, nullptr, table, row + 1, cols, 0, n_pages, lg, err};
  return page_of(p, row, pos);
}

}
