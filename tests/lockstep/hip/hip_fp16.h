// fp16 conversions by the host compiler's type.
#pragma once
#include <cstdint>
#include <cstring>

typedef _Float16 __half;
inline __half __ushort_as_half(uint16_t x) { __half h; memcpy(&h, &x, 2); return h; }
inline uint16_t __half_as_ushort(__half h) { uint16_t x; memcpy(&x, &h, 2); return x; }
inline float __half2float(__half h) { return static_cast<float>(h); }
inline __half __float2half_rn(float f) { return static_cast<__half>(f); }
