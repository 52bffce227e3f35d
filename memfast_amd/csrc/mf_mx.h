// Device helpers of the 4-bit microscaled operands (microscaling.hip, microscaling_grad.hip).
//
// Format.  A block is 32 consecutive values of a row.  With e = max(floor(log2 max|x|) - 2, -126)
// its scale is 2^e, held as the byte e + 127, and a value's code is x / 2^e rounded to nearest even
// on {0, 0.5, 1, 1.5, 2, 3, 4, 6} (sign in bit 3), saturating at 6.  A block that holds a NaN or an
// infinity has scale byte 255 and stands for NaN.  Rows are padded to segments of 256 values
// (128 bytes of codes, the lower half of a byte first, and 8 scale bytes) with zero codes, so that
// every row of codes is whole 128-byte lines and no kernel has a remainder along k.
//
// Scales lie row by row, [n, segs * 8], in tensors that a caller holds, and segment by segment,
// [segs, n rounded up to even, 8], in operands that are quantized within a call: there 32 rows' scales
// of a segment are 256 consecutive bytes. Kernels take them by the strides of a row and a segment.
#pragma once

#include "mf_float.h"

namespace mf {

constexpr int SEG = 256;          // values of a segment
constexpr int SEG_BYTES = 128;    // its codes
constexpr int SEG_SCALES = 8;     // its scale bytes
constexpr u32 NAN_BYTE = 255;

__host__ __device__ inline i64 segments(i64 k) { return (k + SEG - 1) / SEG; }
__host__ __device__ inline i64 even(i64 n) { return (n + 1) / 2 * 2; }

struct Scales {
    const u8 *data;
    i64 row, seg;       // strides
};

__host__ inline Scales scales_by_row(const u8 *data, i64 segs) { return {data, segs * SEG_SCALES, SEG_SCALES}; }
__host__ inline Scales scales_by_segment(const u8 *data, i64 n) {
    return {data, SEG_SCALES, even(n) * SEG_SCALES};
}

// ---- values ----------------------------------------------------------------
// Eight values of a row from column c; zero from column k on.
template <typename T>
__device__ __forceinline__ void load8(const T *row, i64 c, i64 k, bool vec, float (&v)[8]) {
    if (vec && c + 8 <= k) {
        constexpr int P = PIECE<T>;
#pragma unroll
        for (int i = 0; i < 8; i += P) {
            const Piece<T> piece = *reinterpret_cast<const Piece<T> *>(row + c + i);
#pragma unroll
            for (int j = 0; j < P; ++j) v[i + j] = float(piece.v[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < k ? float(row[c + i]) : 0.0f;
    }
}

template <typename T>
__device__ __forceinline__ void store8(T *row, i64 c, i64 k, bool vec, const float (&v)[8]) {
    if (vec && c + 8 <= k) {
        constexpr int P = PIECE<T>;
#pragma unroll
        for (int i = 0; i < 8; i += P) {
            Piece<T> piece;
#pragma unroll
            for (int j = 0; j < P; ++j) piece.v[j] = T(v[i + j]);
            *reinterpret_cast<Piece<T> *>(row + c + i) = piece;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < k) row[c + i] = T(v[i]);
    }
}

// ---- codes -----------------------------------------------------------------
// The largest magnitude's bits: in integer order a NaN is above infinity, and that above the rest.
__device__ __forceinline__ u32 peak8(const float (&v)[8]) {
    u32 peak = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) peak = max(peak, __float_as_uint(v[i]) & 0x7fffffffu);
    return peak;
}

__device__ __forceinline__ u32 scale_byte(u32 peak) {
    const u32 exponent = peak >> 23;
    return exponent == 255u ? NAN_BYTE : max(exponent, 3u) - 2u;
}

// v_cvt_scalef32_pk_fp4_f32 divides by the scale, rounds to nearest even and saturates.
__device__ __forceinline__ u32 codes8(const float (&v)[8], u32 byte) {
    const float scale = __uint_as_float(byte << 23);
    u32 word = 0;
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[0], v[1], scale, 0);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[2], v[3], scale, 1);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[4], v[5], scale, 2);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[6], v[7], scale, 3);
    return byte == NAN_BYTE ? 0u : word;
}

// Eight codes as BF16, exactly: two significant bits, and the scales are BF16's own exponents. The instruction
// takes its scale's exponent field, so that byte 0, which the quantizer does not write, is 2^-127 here
// as in the scaled product (measured: every byte gives the same value in both). Where a code times
// byte 253 or 254 passes FP32's range it is infinite here.
__device__ __forceinline__ v8bf expand8(u32 word, u32 byte) {
    if (byte == NAN_BYTE) {
        const bf16 nan = bf16(__uint_as_float(0x7fc00000u));
        return v8bf{nan, nan, nan, nan, nan, nan, nan, nan};
    }
    const float scale = __uint_as_float(byte << 23);
    const v2bf a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 0);
    const v2bf b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 1);
    const v2bf c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 2);
    const v2bf d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 3);
    return v8bf{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// ---- jobs of one launch ----------------------------------------------------
// Independent passes over matrices share a launch: a job has blocks [first, first + gx * gy). 1 << lanes of a
// block's 256 threads lie along a row's units, the others take further rows.
struct Job {
    u32 first, gx, gy;
    int lanes;
    __device__ __forceinline__ bool mine(u32 block) const { return block - first < gx * gy; }
    __device__ __forceinline__ i64 unit() const {
        return (i64((blockIdx.x - first) % gx) << lanes) + (threadIdx.x & ((1 << lanes) - 1));
    }
    __device__ __forceinline__ i64 row() const {
        return i64((blockIdx.x - first) / gx) * (256 >> lanes) + (threadIdx.x >> lanes);
    }
    __device__ __forceinline__ i64 step() const { return i64(gy) * (256 >> lanes); }
};

// The next job of a launch that has `blocks` blocks so far: `units` of each of `rows` rows.
__host__ inline Job add_job(i64 units, i64 rows, u32 &blocks) {
    int lanes = 3;
    while (lanes < 8 && (i64(1) << lanes) < units) ++lanes;
    const i64 per = 256 >> lanes;
    const i64 gx = (units + (i64(1) << lanes) - 1) >> lanes;
    const i64 most = gx < 32768 ? 262144 / gx : 8;      // then a thread takes several rows
    i64 gy = (rows + per - 1) / per;
    if (gy > most) gy = most;
    const Job job{blocks, u32(gx), u32(gy), lanes};
    blocks += u32(gx * gy);
    return job;
}

// ---- copies ahead of the matrix cores -------------------------------------
// Waits until at most N of this wave's vector memory operations are outstanding and its LDS reads
// have arrived, then for the other waves: every copy before those N is then in LDS, and the buffer
// that was read before may be written. The copies are inline assembly, which the compiler neither
// counts nor orders against its own LDS reads; hence the empty assembly on both sides.
template <int N> __device__ __forceinline__ void wait_stage() {
    static_assert(N < 64, "vmcnt has six bits");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4);     // lgkmcnt 0, expcnt any
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

__device__ __forceinline__ u32 lds_address(const u8 *p) {
    return u32(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) u8 *)p));
}

}  // namespace mf
