// Argument checks that C entries share.
#pragma once

namespace {
// one of these required pointers is missing: the kernel would read or write address 0
template <typename... P> inline bool any_null(P... p) { return ((p == nullptr) || ...); }
}  // namespace
