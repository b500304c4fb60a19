// A runtime context without a device, for tests of argument checks: the entry points look at their arguments before they make any
// CUDA call, so a call that has to be refused never reaches the GPU.  Storages are registered with rb_import under made-up addresses.
#include "common.cuh"

extern "C" __attribute__((visibility("default"))) rb_ctx* host_context() {
    rb_ctx* ctx = new rb_ctx();
    ctx->sm_count = 148;
    return ctx;
}
extern "C" __attribute__((visibility("default"))) void host_context_free(rb_ctx* ctx) { delete ctx; }
