// The floating types that the microscaled and distillation kernels read and write, loads and stores of
// whole 16-byte pieces of them, and what their host sides share.
#pragma once

#include "mf_device.h"

namespace mf {

typedef __bf16 bf16;
typedef _Float16 f16;

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef u32 v4u __attribute__((ext_vector_type(4)));
typedef u32 v2u __attribute__((ext_vector_type(2)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef bf16 v8bf __attribute__((ext_vector_type(8)));
typedef bf16 v2bf __attribute__((ext_vector_type(2)));

// Values of T in 16 bytes.
template <typename T> constexpr int PIECE = 16 / int(sizeof(T));

template <typename T> struct alignas(16) Piece {
    T v[PIECE<T>];
};

// Calls f(T{}) with the element type of an MF_F32 / MF_BF16 / MF_F16 code.
template <typename F> __host__ int with_type(int32_t type, F f) {
    switch (type) {
    case MF_F32: return f(float{});
    case MF_BF16: return f(bf16{});
    default: return f(f16{});
    }
}

__host__ inline int type_bytes(int32_t type) { return type == MF_F32 ? 4 : 2; }
__host__ inline bool known_type(int32_t type) { return type >= MF_F32 && type <= MF_F16; }

// api.hip
int fail(int code, const char *fmt, ...);
int check_launch(const char *what);
bool aligned(const void *p, uintptr_t bytes);

// Dynamic LDS that passes 64 KiB, with up to 16 KiB of the kernel's own beside it, has to be asked for: on
// the kernel's current device, so at every launch.
template <typename K> __host__ int allow_lds(K kernel, i64 bytes) {
    if (bytes <= 48 << 10) return MF_OK;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
    return e == hipSuccess
               ? MF_OK
               : fail(MF_E_RESOURCE, "LDS of %lld bytes: %s", (long long)bytes, hipGetErrorString(e));
}

}  // namespace mf
