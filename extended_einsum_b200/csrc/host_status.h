// The message behind xe_last_error_string, shared by the host side of every translation unit.
#pragma once

#include "../../include/xe_b200.h"

namespace xe {

// Records the message for this host thread and returns `code`.
__attribute__((format(printf, 2, 3), visibility("hidden"))) xe_status fail(xe_status code, const char* format, ...);

}  // namespace xe
