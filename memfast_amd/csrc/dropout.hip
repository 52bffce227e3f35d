// Dropout from a counter-based generator: the mask is made anew wherever it is needed and never stored.
//
// Value i is dropped where the 16-bit number i % 8 of Philox 4x32-10 (Salmon, Moraes, Dror and Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", 2011) for the counter (i / 8, event) and the key
// `seed` is below `dropped`, so one in 65536 is the step of the probability, and kept values are divided
// by the exact share of those that are kept.  The generator of the devices' noise, one avalanche hash of
// 32 bits, would give masks that are the same bits in another order for every seed and event.
#include <algorithm>

#include "mf_float.h"

namespace mf {

struct DropoutArgs {
    const void *x, *residual;   // [n]; residual may be nullptr
    i64 n;
    u32 dropped;                // of 65536
    float scale;
    u64 seed, event;
    const i64 *event_at;        // or nullptr; the event is read here then
    void *y;
};

__device__ __forceinline__ void philox(u32 (&c)[4], u32 k0, u32 k1) {
#pragma unroll
    for (int turn = 0; turn < 10; ++turn) {
        const u64 left = u64(c[0]) * 0xD2511F53u, right = u64(c[2]) * 0xCD9E8D57u;
        c[0] = u32(right >> 32) ^ c[1] ^ k0;
        c[1] = u32(right);
        c[2] = u32(left >> 32) ^ c[3] ^ k1;
        c[3] = u32(left);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
}

// A lane takes the eight values of one block of the generator. PIECES: whole 16-byte loads and stores. Bound by its
// bytes: 8192 x 4096 BF16 in 26 us (134 MB, 5.1 TB/s), with a residual in 36 (201 MB); the generator's ten rounds
// and the rest are 300 vector instructions a lane, which take 63% of that.
template <typename T, bool PIECES> __global__ __launch_bounds__(256) void k_dropout(const DropoutArgs a) {
    constexpr int N = PIECE<T>;
    const T *x = static_cast<const T *>(a.x), *residual = static_cast<const T *>(a.residual);
    T *y = static_cast<T *>(a.y);
    const u64 event = a.event_at ? u64(*a.event_at) : a.event;
    const i64 blocks = (a.n + 7) / 8;
    for (i64 block = i64(blockIdx.x) * 256 + threadIdx.x; block < blocks; block += i64(gridDim.x) * 256) {
        const i64 first = block * 8;
        const bool whole = PIECES && first + 8 <= a.n;
        alignas(16) T v[8], r[8];
        if (whole) {
#pragma unroll
            for (int i = 0; i < 8; i += N) {
                *reinterpret_cast<Piece<T> *>(v + i) = *reinterpret_cast<const Piece<T> *>(x + first + i);
                if (residual)
                    *reinterpret_cast<Piece<T> *>(r + i) =
                        *reinterpret_cast<const Piece<T> *>(residual + first + i);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const i64 at = min(first + i, a.n - 1);
                v[i] = x[at];
                if (residual) r[i] = residual[at];
            }
        }
        u32 c[4] = {u32(block), u32(u64(block) >> 32), u32(event), u32(event >> 32)};
        philox(c, u32(a.seed), u32(a.seed >> 32));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const u32 number = i % 2 ? c[i / 2] >> 16 : c[i / 2] & 0xffffu;
            const float before = residual ? float(r[i]) : 0.0f;
            // A dropped value is gone whatever it was, an infinity or NaN too.
            const float kept = residual ? fmaf(float(v[i]), a.scale, before) : float(v[i]) * a.scale;
            v[i] = rounded<T>(number < a.dropped ? before : kept);
        }
        if (whole) {
#pragma unroll
            for (int i = 0; i < 8; i += N)
                *reinterpret_cast<Piece<T> *>(y + first + i) = *reinterpret_cast<Piece<T> *>(v + i);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (first + i < a.n) y[first + i] = v[i];
        }
    }
}

}  // namespace mf

using namespace mf;

extern "C" int mf_dropout(const void *x, int32_t type, int64_t n, const void *residual, uint32_t dropped,
                          uint64_t seed, uint64_t event, const int64_t *event_at, void *y, void *stream) {
    if (!x || !y || !known_type(type) || n < 1 || n > i64(1) << 40 || dropped > 65536)
        return fail(MF_E_INVALID, "invalid dropout arguments");
    const uintptr_t one = type_bytes(type);
    if (!aligned(x, one) || !aligned(residual, one) || !aligned(y, one) || !aligned(event_at, 8))
        return fail(MF_E_INVALID, "dropout operands are not aligned to their types");
    const float scale = dropped == 65536 ? 0.0f : float(65536.0 / double(65536 - dropped));
    const DropoutArgs args{x, residual, n, dropped, scale, seed, event, event_at, y};
    const bool pieces = aligned(x, 16) && aligned(residual, 16) && aligned(y, 16);
    const u32 grid = u32(std::min<i64>((n + 2047) / 2048, i64(1) << 20));
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        hipLaunchKernelGGL((pieces ? k_dropout<T, true> : k_dropout<T, false>), dim3(grid), dim3(256), 0,
                           static_cast<hipStream_t>(stream), args);
        return check_launch("dropout");
    });
}

extern "C" int mf_capture_id(void *stream, uint64_t *id) {
    if (!id) return fail(MF_E_INVALID, "no place for a capture's number");
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long number = 0;
    const hipError_t e = hipStreamGetCaptureInfo(static_cast<hipStream_t>(stream), &status, &number);
    if (e != hipSuccess) return fail(MF_E_HIP, "capture of a stream: %s", hipGetErrorString(e));
    *id = status == hipStreamCaptureStatusActive ? u64(number) : 0;
    return MF_OK;
}
