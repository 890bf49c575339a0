#pragma once

#include <cstdint>

struct __half {
    uint16_t bits;
};
typedef __half half;
