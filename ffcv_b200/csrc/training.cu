// Errors of the training step's entry points.
#include "training.h"

#include <stdarg.h>

namespace ffcvb {

namespace {
thread_local char t_error[256] = "";
}

int training_fail(int code, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(t_error, sizeof(t_error), fmt, ap);
    va_end(ap);
    return code;
}

} // namespace ffcvb

extern "C" const char *ffcvb_training_error(void) { return ffcvb::t_error; }
