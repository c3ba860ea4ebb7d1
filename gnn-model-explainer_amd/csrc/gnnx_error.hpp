// gnnx_error.hpp — the error text behind gnnx_last_error(), shared by the library's translation units.
#pragma once

namespace gnnx {
__attribute__((visibility("hidden"))) int set_error(const char* text) noexcept;   // the calling thread's text; returns 1
}
