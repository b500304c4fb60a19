// Host build of the 8-bit linear's choice of kernel (rust_ascend_b200/csrc/linear_plan.h) for CPU tests.
#include "linear_plan.h"
extern "C" void host_linear_plan(uint32_t m, uint32_t n, uint32_t k, uint32_t sms, uint32_t pairs, int limited, uint32_t* out3) {
    const rb_linear_plan p = rb_linear_plan_of(m, n, k, sms, pairs, limited != 0);
    out3[0] = p.tokens; out3[1] = p.parts; out3[2] = p.rows;
}
