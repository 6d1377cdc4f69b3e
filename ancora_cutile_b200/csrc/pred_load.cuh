// Predicated loads that leave the registers alone where `on` is false.  They are single instructions
// because the value of an `if` is merged by a register move that waits for the load: written with
// branches, loops that fetch ahead or guard their last round had one load in flight per warp.
#pragma once
#include <stdint.h>

__device__ __forceinline__ void ld_v4(uint32_t &a, uint32_t &b, uint32_t &c, uint32_t &d, const void *p, bool on) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %5, 0;\n\t@q ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
               : "+r"(a), "+r"(b), "+r"(c), "+r"(d)
               : "l"(p), "r"((uint32_t)on)
               : "memory");
}
// 32 bytes, 32-byte aligned
__device__ __forceinline__ void ld_v8(uint32_t (&r)[8], const void *p, bool on) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %9, 0;\n\t@q ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\t}"
      : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
      : "l"(p), "r"((uint32_t)on)
      : "memory");
}
__device__ __forceinline__ void ld_1(uint32_t &a, const void *p, bool on) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %2, 0;\n\t@q ld.global.u32 %0, [%1];\n\t}"
               : "+r"(a)
               : "l"(p), "r"((uint32_t)on)
               : "memory");
}
// 16 bits, zero-extended
__device__ __forceinline__ void ld_h(uint32_t &a, const void *p, bool on) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %2, 0;\n\t@q ld.global.u16 %0, [%1];\n\t}"
               : "+r"(a)
               : "l"(p), "r"((uint32_t)on)
               : "memory");
}
// 32 bytes, 32-byte aligned
__device__ __forceinline__ void st_v8(void *p, const float (&x)[8]) {
  asm volatile("st.global.v8.f32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]),
               "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]), "l"(p)
               : "memory");
}
