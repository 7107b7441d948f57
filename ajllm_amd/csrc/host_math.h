// Whole numbers on the host.
#pragma once

namespace {

inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

}  // namespace
