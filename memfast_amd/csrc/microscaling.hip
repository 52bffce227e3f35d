// 4-bit microscaled floating point: quantization in blocks of 32, the product of two such
// operands, and its gradients.
//
// Format.  A block is 32 consecutive values of a row.  With e = max(floor(log2 max|x|) - 2, -126)
// its scale is 2^e, held as the byte e + 127, and a value's code is x / 2^e rounded to nearest even
// on {0, 0.5, 1, 1.5, 2, 3, 4, 6} (sign in bit 3), saturating at 6.  A block that holds a NaN or an
// infinity has scale byte 255 and stands for NaN.  Rows are padded to segments of 256 values
// (128 bytes of codes, the lower half of a byte first, and 8 scale bytes) with zero codes, so that
// every row of codes is whole 128-byte lines and no kernel has a remainder along k.
//
// Product.  y = Q(x) Q(W)^T + b runs on v_mfma_scale_f32_*_f8f6f4, which takes one block of a row
// (16 bytes) and its scale byte per lane, so both operands go from memory to the matrix cores as
// they are.  Sums are FP32.
//
// Gradients, straight through the quantizers: dx = dy Q(W), dw = dy^T Q(x), db = sum_n dy.  They
// contract over the rows of the 4-bit operand, whose scales change from row to row, so the block
// scales of the matrix instruction cannot carry them.  A code times its scale is exact in BF16
// (two significant bits), so the 4-bit operand is expanded to BF16 in LDS, and dy enters as
// BF16 terms whose sum is its value exactly: one for BF16, two for FP16, three for FP32.
#include <algorithm>
#include <type_traits>

#include "mf_float.h"

namespace mf {

constexpr int SEG = 256;          // values of a segment
constexpr int SEG_BYTES = 128;    // its codes
constexpr int SEG_SCALES = 8;     // its scale bytes
constexpr u32 NAN_BYTE = 255;

__host__ __device__ inline i64 segments(i64 k) { return (k + SEG - 1) / SEG; }

// The FP32 scale of a scale byte (NaN for 255: 0x7fc00000 and 255 << 23 share their exponent).
__device__ __forceinline__ float scale_of(u32 byte) {
    return __uint_as_float(byte == NAN_BYTE ? 0x7fc00000u : byte << 23);
}

// ---------------------------------------------------------------------------
// Quantization
// ---------------------------------------------------------------------------
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

// One lane quantizes eight values and four neighbours share a block.  1 << lanes lanes lie along a
// row, the others take further rows. Scales go to [n, segs * 8], or to [segs, n, 8] if `turned`.
template <typename T>
__global__ __launch_bounds__(256) void k_mx_quantize(const T *x, i64 n, i64 k, i64 ldx, bool vec,
                                                     int lanes, bool turned, u8 *codes,
                                                     u8 *scales) {
    const i64 segs = segments(k), units = segs * 32;
    const i64 unit = (i64(blockIdx.x) << lanes) + (threadIdx.x & ((1 << lanes) - 1));
    const i64 step = i64(gridDim.y) * (256 >> lanes);
    if (unit >= units) return;
    for (i64 r = i64(blockIdx.y) * (256 >> lanes) + (threadIdx.x >> lanes); r < n; r += step) {
        float v[8];
        load8(x + r * ldx, unit * 8, k, vec, v);
        u32 peak = peak8(v);
        peak = max(peak, u32(__shfl_xor(int(peak), 1)));
        peak = max(peak, u32(__shfl_xor(int(peak), 2)));
        const u32 byte = scale_byte(peak);
        reinterpret_cast<u32 *>(codes + r * segs * SEG_BYTES)[unit] = codes8(v, byte);
        if ((unit & 3) == 0)
            scales[turned ? (unit / 32 * n + r) * SEG_SCALES + (unit / 4 & 7)
                          : r * segs * SEG_SCALES + unit / 4] = u8(byte);
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

__device__ __forceinline__ void values8(u32 word, float scale, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const u32 code = word >> (4 * i), m = code & 7u;
        // 0, 0.5, 1, 1.5, 2, 3, 4, 6
        const float size = m < 4u ? 0.5f * float(m) : float((2u | (m & 1u)) << ((m - 4u) >> 1));
        v[i] = (code & 8u ? -size : size) * scale;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void k_mx_dequantize(const u8 *codes, const u8 *scales, i64 n,
                                                       i64 k, bool vec, int lanes, T *out) {
    const i64 segs = segments(k), units = (k + 7) / 8;
    const i64 unit = (i64(blockIdx.x) << lanes) + (threadIdx.x & ((1 << lanes) - 1));
    const i64 step = i64(gridDim.y) * (256 >> lanes);
    if (unit >= units) return;
    for (i64 r = i64(blockIdx.y) * (256 >> lanes) + (threadIdx.x >> lanes); r < n; r += step) {
        float v[8];
        values8(reinterpret_cast<const u32 *>(codes + r * segs * SEG_BYTES)[unit],
                scale_of(scales[r * segs * SEG_SCALES + unit / 4]), v);
        store8(out + r * k, unit * 8, k, vec, v);
    }
}

// ---------------------------------------------------------------------------
// Product
// ---------------------------------------------------------------------------
// Bytes h, 2 + h, 4 + h and 6 + h of a segment's eight scale bytes: the scales of the blocks that
// lanes of half h hold in the segment's four 64-value steps.
__device__ __forceinline__ u32 half_scales(v2u s, int h) {
    return __builtin_amdgcn_perm(s.y, s.x, h ? 0x07050301u : 0x06040200u);
}

template <int STEP>
__device__ __forceinline__ v16f mfma_step(v4u a, v4u b, v16f c, u32 sa, u32 sb) {
    const v8i av = {int(a.x), int(a.y), int(a.z), int(a.w), 0, 0, 0, 0};
    const v8i bv = {int(b.x), int(b.y), int(b.z), int(b.w), 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, c, 4, 4, STEP, int(sa), STEP,
                                                           int(sb));
}

struct MxArgs {
    const u8 *xc, *xs;      // codes [n, segs * 128], scales [segs, n, 8]
    const u8 *wc, *ws;      // codes [o, segs * 128], scales [o, segs * 8] (tiles: [segs, o, 8])
    const void *x;          // k_mx_few<..., true>: the input itself, rows ldx apart
    i64 ldx, k;
    bool vec;
    const void *bias;       // [o] or nullptr
    void *out;              // [n, o]
    i64 n, o, segs;
};

// ---- few rows --------------------------------------------------------------
// Up to 64 rows of x: the weight's bytes bound it, so each is loaded once, straight into the operand
// registers. A workgroup takes 16 rows of W; its eight waves split the segments and add their
// sums in LDS in the order of the waves. QUANTIZE: the workgroup quantizes x into LDS itself, while
// its first weights are on their way, which saves a launch; else Q(x) is read from the cache.
constexpr int FEW_WAVES = 8, FEW_TILE = 16;

__device__ __forceinline__ v4f mfma_few(v4u a, v4u b, v4f c, u32 sa, u32 sb) {
    const v8i av = {int(a.x), int(a.y), int(a.z), int(a.w), 0, 0, 0, 0};
    const v8i bv = {int(b.x), int(b.y), int(b.z), int(b.w), 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 0, int(sa), 0, int(sb));
}

__host__ __device__ inline i64 few_pitch(i64 segs) { return segs * SEG_BYTES + 16; }

__host__ inline i64 few_lds(i64 n, i64 segs) {
    return n * few_pitch(segs) + n * segs * SEG_SCALES;
}

template <typename T, int NT, bool QUANTIZE>
__global__ __launch_bounds__(64 * FEW_WAVES) void k_mx_few(const MxArgs a) {
    extern __shared__ __align__(16) u8 staged[];
    __shared__ float part[FEW_WAVES][NT][FEW_TILE * FEW_TILE];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = lane & 15, block = lane >> 4;
    const i64 o0 = i64(blockIdx.x) * FEW_TILE;
    const i64 per = (a.segs + FEW_WAVES - 1) / FEW_WAVES;
    const i64 first = min(wave * per, a.segs), last = min(first + per, a.segs);
    // Rows past the end read the last row; their results are not stored.
    const i64 o = min(o0 + row, a.o - 1);
    const u8 *wc = a.wc + o * a.segs * SEG_BYTES + block * 16, *ws = a.ws + o * a.segs * SEG_SCALES;

    v4u w[2];
    v2u sw;
    auto load_weight = [&](i64 s) {
        w[0] = *reinterpret_cast<const v4u *>(wc + s * SEG_BYTES);
        w[1] = *reinterpret_cast<const v4u *>(wc + s * SEG_BYTES + 64);
        sw = *reinterpret_cast<const v2u *>(ws + s * SEG_SCALES);
    };
    if (first < last) load_weight(first);

    const i64 pitch = few_pitch(a.segs);
    u8 *const staged_scales = staged + a.n * pitch;
    if (QUANTIZE) {
        const i64 units = a.segs * 32;
        for (i64 r = 0; r < a.n; ++r)
            for (i64 unit = tid; unit < units; unit += 64 * FEW_WAVES) {
                float v[8];
                load8(static_cast<const T *>(a.x) + r * a.ldx, unit * 8, a.k, a.vec, v);
                u32 peak = peak8(v);
                peak = max(peak, u32(__shfl_xor(int(peak), 1)));
                peak = max(peak, u32(__shfl_xor(int(peak), 2)));
                const u32 byte = scale_byte(peak);
                reinterpret_cast<u32 *>(staged + r * pitch)[unit] = codes8(v, byte);
                if ((unit & 3) == 0)
                    staged_scales[r * a.segs * SEG_SCALES + unit / 4] = u8(byte);
            }
        __syncthreads();
    }

    v4f acc[NT] = {};
    for (i64 s = first; s < last; ++s) {
        const v4u w0 = w[0], w1 = w[1];
        const v2u scale = sw;
        if (s + 1 < last) load_weight(s + 1);
        const u32 sw0 = scale.x >> (8 * block), sw1 = scale.y >> (8 * block);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const i64 r = min(i64(16 * t + row), a.n - 1);
            const u8 *xc = QUANTIZE ? staged + r * pitch : a.xc + r * a.segs * SEG_BYTES;
            const u8 *xs = QUANTIZE ? staged_scales + r * a.segs * SEG_SCALES + s * SEG_SCALES
                                    : a.xs + (s * a.n + r) * SEG_SCALES;
            const v4u x0 = *reinterpret_cast<const v4u *>(xc + s * SEG_BYTES + block * 16);
            const v4u x1 = *reinterpret_cast<const v4u *>(xc + s * SEG_BYTES + 64 + block * 16);
            const v2u sx = *reinterpret_cast<const v2u *>(xs);
            acc[t] = mfma_few(x0, w0, acc[t], sx.x >> (8 * block), sw0);
            acc[t] = mfma_few(x1, w1, acc[t], sx.y >> (8 * block), sw1);
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[wave][t][(4 * block + i) * FEW_TILE + row] = acc[t][i];
    __syncthreads();
    for (int e = tid; e < NT * FEW_TILE * FEW_TILE; e += 64 * FEW_WAVES) {
        const int t = e / (FEW_TILE * FEW_TILE), at = e % (FEW_TILE * FEW_TILE);
        const i64 n = 16 * t + at / FEW_TILE, c = o0 + at % FEW_TILE;
        if (n >= a.n || c >= a.o) continue;
        float sum = part[0][t][at];
#pragma unroll
        for (int w = 1; w < FEW_WAVES; ++w) sum += part[w][t][at];
        if (a.bias) sum += float(static_cast<const T *>(a.bias)[c]);
        static_cast<T *>(a.out)[n * a.o + c] = T(sum);
    }
}

// ---- many rows -------------------------------------------------------------
// WN x WO waves of TN x TO tiles of 32 x 32. A stage is one segment (128 bytes) of every row of the
// tile, copied to LDS without passing through registers, one stage ahead of the matrix cores.
// The 16-byte pieces of row r lie rotated by r & 7, so that the eight rows that a read serves at
// once are in different banks. Scales come segment by segment ([segs, rows, 8]): a wave reads those
// of 32 rows as 256 consecutive bytes, one segment ahead, into registers.
template <typename T, int WN, int WO, int TN, int TO>
__global__ __launch_bounds__(64 * WN * WO) void k_mx_tile(const MxArgs a) {
    constexpr int BN = 32 * WN * TN, BO = 32 * WO * TO, WAVES = WN * WO;
    constexpr int COPIES = (BN + BO) / 8 / WAVES;   // of 8 rows, by each wave
    static_assert((BN + BO) % (8 * WAVES) == 0, "whole copies");
    extern __shared__ __align__(16) u8 staged[];      // [2][BN + BO][128]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int half = lane >> 5, row = lane & 31;
    u32 tx, ty;
    xcd_tile(blockIdx.x, u32((a.n + BN - 1) / BN), u32((a.o + BO - 1) / BO), tx, ty);
    const i64 n0 = i64(tx) * BN, o0 = i64(ty) * BO;
    const i64 pitch = a.segs * SEG_BYTES;

    // Where this lane's copies come from, eight rows of one operand each: rows past the end read
    // the last row.
    const int first_copy = __builtin_amdgcn_readfirstlane(wave * COPIES);
    const u8 *const x0 = a.xc + n0 * pitch, *const w0 = a.wc + o0 * pitch;
    u32 offset[COPIES];
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
        const int r = (first_copy + i) * 8 + (lane >> 3);
        const i64 at = r < BN ? min(i64(r), a.n - n0 - 1) : min(i64(r - BN), a.o - o0 - 1);
        offset[i] = u32(at * pitch) + u32(((lane & 7) ^ (lane >> 3)) * 16);
    }
    const u32 lds = u32(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) u8 *)staged));
    auto copy = [&](i64 s, int buffer) {
#pragma unroll
        for (int i = 0; i < COPIES; ++i) {
            const int r = (first_copy + i) * 8;
            lds_dma_16((r < BN ? x0 : w0) + s * SEG_BYTES + offset[i],
                       __builtin_amdgcn_readfirstlane(lds + (buffer * (BN + BO) + r) * SEG_BYTES));
        }
    };

    const int wn = (wave / WO) * TN * 32, wo = (wave % WO) * TO * 32;
    u32 xat[TN], wat[TO];       // scale offsets of this lane's rows in a segment
#pragma unroll
    for (int i = 0; i < TN; ++i) xat[i] = u32(min(n0 + wn + 32 * i + row, a.n - 1)) * SEG_SCALES;
#pragma unroll
    for (int j = 0; j < TO; ++j) wat[j] = u32(min(o0 + wo + 32 * j + row, a.o - 1)) * SEG_SCALES;
    v2u xs[TN], ws[TO];
    auto load_scales = [&](i64 s) {
#pragma unroll
        for (int i = 0; i < TN; ++i)
            xs[i] = *reinterpret_cast<const v2u *>(a.xs + s * a.n * SEG_SCALES + xat[i]);
#pragma unroll
        for (int j = 0; j < TO; ++j)
            ws[j] = *reinterpret_cast<const v2u *>(a.ws + s * a.o * SEG_SCALES + wat[j]);
    };

    v16f acc[TN][TO] = {};
    copy(0, 0);
    load_scales(0);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    for (i64 s = 0; s < a.segs; ++s) {
        u32 sx[TN], sw[TO];
#pragma unroll
        for (int i = 0; i < TN; ++i) sx[i] = half_scales(xs[i], half);
#pragma unroll
        for (int j = 0; j < TO; ++j) sw[j] = half_scales(ws[j], half);
        if (s + 1 < a.segs) {
            copy(s + 1, int(s + 1) & 1);
            load_scales(s + 1);
        }
        const u8 *xt = staged + (int(s) & 1) * (BN + BO) * SEG_BYTES + (wn + row) * SEG_BYTES;
        const u8 *wt = staged + (int(s) & 1) * (BN + BO) * SEG_BYTES + (BN + wo + row) * SEG_BYTES;
        auto step = [&](auto number) {
            constexpr int STEP = decltype(number)::value;
            const int piece = ((2 * STEP + half) ^ (row & 7)) * 16;
            v4u fx[TN], fw[TO];
#pragma unroll
            for (int i = 0; i < TN; ++i)
                fx[i] = *reinterpret_cast<const v4u *>(xt + i * 32 * SEG_BYTES + piece);
#pragma unroll
            for (int j = 0; j < TO; ++j)
                fw[j] = *reinterpret_cast<const v4u *>(wt + j * 32 * SEG_BYTES + piece);
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int j = 0; j < TO; ++j)
                    acc[i][j] = mfma_step<STEP>(fx[i], fw[j], acc[i][j], sx[i], sw[j]);
        };
        step(std::integral_constant<int, 0>{});
        step(std::integral_constant<int, 1>{});
        step(std::integral_constant<int, 2>{});
        step(std::integral_constant<int, 3>{});
        // The copies are not in the compiler's count of outstanding loads.
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
    }
    T *out = static_cast<T *>(a.out);
#pragma unroll
    for (int j = 0; j < TO; ++j) {
        const i64 c = o0 + wo + 32 * j + row;
        if (c >= a.o) continue;
        const float bias = a.bias ? float(static_cast<const T *>(a.bias)[c]) : 0.0f;
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const i64 r = n0 + wn + 32 * i + 8 * (e / 4) + 4 * half + (e & 3);
                if (r < a.n) out[r * a.o + c] = T(acc[i][j][e] + bias);
            }
    }
}

// Scales [rows, segs * 8] as [segs, rows, 8].
__global__ __launch_bounds__(256) void k_mx_turn_scales(const v2u *in, i64 rows, i64 segs, v2u *out) {
    const i64 r = i64(blockIdx.x) * 256 + threadIdx.x;
    if (r < rows) out[blockIdx.y * rows + r] = in[r * segs + blockIdx.y];
}

// ---------------------------------------------------------------------------
// Gradients
// ---------------------------------------------------------------------------
constexpr int GRAD_STEP = 64;     // of the contraction in one stage

struct GradArgs {
    const bf16 *a;      // dy terms: plane t at a + t * plane, rows of lda values
    i64 plane, lda;
    i64 width;          // values of a row that may be read, a multiple of 8
    int terms;
    const bf16 *b;      // the 4-bit operand expanded, [depth in whole steps, cols in segments]
    i64 ldb;
    i64 rows, cols;     // of the result
    i64 depth;          // contraction
    void *out;          // [rows, cols]
};

// dy [n, o] as `terms` planes of BF16, [terms][rows][cols] with zeros past n and o: the terms add
// up to the value exactly (each takes eight significant bits by truncation, which also keeps the
// largest finite values finite).
template <typename T>
__global__ __launch_bounds__(256) void k_mx_terms(const T *dy, i64 n, i64 o, i64 ldy, int terms,
                                                  i64 rows, i64 cols, bf16 *out) {
    const i64 c = i64(blockIdx.x) * 256 + threadIdx.x;
    if (c >= cols) return;
    for (i64 r = blockIdx.y; r < rows; r += gridDim.y) {
        float rest = r < n && c < o ? float(dy[r * ldy + c]) : 0.0f;
        const bool finite = (__float_as_uint(rest) & 0x7f800000u) != 0x7f800000u;
        for (int t = 0; t < terms; ++t) {
            // A NaN or an infinity is its own first term.
            const float term = finite ? __uint_as_float(__float_as_uint(rest) & 0xffff0000u)
                                      : (t == 0 ? rest : 0.0f);
            out[(i64(t) * rows + r) * cols + c] = bf16(term);
            if (finite) rest -= term;
        }
    }
}

// Codes [n, segs * 128] as BF16 [rows, segs * 256], zeros past n; scales [n, segs * 8], or
// [segs, n, 8] if `turned`. A lane expands eight values.
__global__ __launch_bounds__(256) void k_mx_expand(const u32 *codes, const u8 *scales, i64 n, i64 segs,
                                                   bool turned, i64 rows, bf16 *out) {
    const i64 unit = i64(blockIdx.x) * 256 + threadIdx.x;
    if (unit >= segs * 32) return;
    for (i64 r = blockIdx.y; r < rows; r += gridDim.y) {
        v8bf v = {};
        if (r < n) {
            const u32 word = codes[r * segs * 32 + unit];
            const float scale =
                scale_of(scales[turned ? (unit / 32 * n + r) * SEG_SCALES + (unit / 4 & 7)
                                       : r * segs * SEG_SCALES + unit / 4]);
            float x[8];
            values8(word, scale, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = bf16(x[i]);
        }
        *reinterpret_cast<v8bf *>(out + (r * segs * 32 + unit) * 8) = v;
    }
}

typedef __attribute__((address_space(3))) v4s *lds_v4s;

// The values of rows r .. r + 3 and r + 4 .. r + 7 of a lane's column, from the address of the four
// columns' piece that this lane supplies of row r + (lane & 15) / 4.
__device__ __forceinline__ v8bf transposed(const u8 *p, int four_rows) {
    union {
        v4s s[2];
        v8bf v;
    } u;
    u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(p));
    u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(p + four_rows));
    return u.v;
}

// How far the 16-byte pieces of row r lie rotated in LDS, in rows of that many pieces: four
// consecutive rows' reads of 64 bytes are then in different banks.
template <int PIECES> __device__ __forceinline__ int rotation(int r) {
    static_assert(PIECES == 8 || PIECES == 16 || PIECES == 32, "the rotation stays within the row");
    return PIECES == 8 ? 4 * (r >> 1 & 1) : 4 * (r & 3);
}

// out[m, c] = sum_t sum_d A_t[m, d] B[d, c], WM x WC waves of TM x TC tiles of 32 x 32, 64 of the
// contraction a stage, copied to LDS one stage ahead without passing through registers.
// DEPTH_ROWS: A's rows run along the contraction (dw: A is dy^T); else along m (dx). Operands whose rows
// run along the contraction are read transposed, four rows of 16 columns by 16 lanes.
template <typename T, bool DEPTH_ROWS, int WM, int WC, int TM, int TC>
__global__ __launch_bounds__(64 * WM * WC) void k_mx_grad(const GradArgs a) {
    constexpr int BM = 32 * WM * TM, BC = 32 * WC * TC, WAVES = WM * WC;
    constexpr int A_BYTES = BM * GRAD_STEP * 2, STAGE = (BM + BC) * GRAD_STEP * 2;
    constexpr int COPIES = STAGE / 1024 / WAVES;
    static_assert(STAGE % (1024 * WAVES) == 0 && A_BYTES % 1024 == 0, "whole copies");
    extern __shared__ __align__(16) u8 staged[];    // [2][A, B]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    u32 tx, ty;
    xcd_tile(blockIdx.x, u32((a.rows + BM - 1) / BM), u32((a.cols + BC - 1) / BC), tx, ty);
    const i64 m0 = i64(tx) * BM, c0 = i64(ty) * BC;

    const int first_copy = __builtin_amdgcn_readfirstlane(wave * COPIES);
    u32 offset[COPIES];
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
        const int at = (first_copy + i) * 1024;
        if (at < A_BYTES && !DEPTH_ROWS) {      // rows of 64 values, 8 pieces rotated by the row
            const int piece = at / 16 + lane, r = piece >> 3;
            offset[i] = u32(min(i64(r), a.rows - m0 - 1) * a.lda * 2) + u32(((piece ^ r) & 7) * 16);
        } else if (at < A_BYTES) {
            constexpr int PIECES = BM / 8;
            const int piece = at / 16 + lane, r = piece / PIECES;
            const int p = piece % PIECES ^ rotation<PIECES>(r);
            offset[i] = u32(r * a.lda * 2) + u32(min(m0 + p * 8, a.width - 8) - m0) * 2;
        } else {
            constexpr int PIECES = BC / 8;
            const int piece = (at - A_BYTES) / 16 + lane, r = piece / PIECES;
            offset[i] = u32(r * a.ldb * 2) + u32((piece % PIECES ^ rotation<PIECES>(r)) * 16);
        }
    }
    const u32 lds = u32(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) u8 *)staged));
    const i64 steps = (a.depth + GRAD_STEP - 1) / GRAD_STEP, stages = steps * a.terms;
    int term = a.terms - 1;     // the smallest terms first
    i64 step = 0;               // of the next copy
    auto copy = [&](int buffer) {
        const bf16 *plane = a.a + term * a.plane;
        const u8 *a0 = reinterpret_cast<const u8 *>(
            DEPTH_ROWS ? plane + step * GRAD_STEP * a.lda + m0 : plane + m0 * a.lda + step * GRAD_STEP);
        const u8 *b0 = reinterpret_cast<const u8 *>(a.b + step * GRAD_STEP * a.ldb + c0);
#pragma unroll
        for (int i = 0; i < COPIES; ++i) {
            const int at = (first_copy + i) * 1024;
            lds_dma_16((at < A_BYTES ? a0 : b0) + offset[i],
                       __builtin_amdgcn_readfirstlane(lds + buffer * STAGE + at));
        }
        if (++step == steps) {
            step = 0;
            --term;
        }
    };

    // Where this lane's fragments start in a stage.
    const int wm = (wave / WC) * TM * 32, wc = (wave % WC) * TC * 32;
    const int i16 = lane & 15, side = lane >> 4 & 1, half = lane >> 5;
    int at_a[TM], at_b[TC];
    auto turned_at = [&](int col, auto width) {
        constexpr int PIECES = decltype(width)::value / 8;
        const int r = 8 * half + (i16 >> 2), piece = (col + 16 * side) / 8 + (i16 & 3) / 2;
        return r * PIECES * 16 + (piece ^ rotation<PIECES>(r)) * 16 + (i16 & 1) * 8;
    };
    const std::integral_constant<int, BM> bm{};
    const std::integral_constant<int, BC> bc{};
#pragma unroll
    for (int i = 0; i < TM; ++i)
        at_a[i] = DEPTH_ROWS ? turned_at(wm + 32 * i, bm) : (wm + 32 * i + (lane & 31)) * GRAD_STEP * 2;
#pragma unroll
    for (int j = 0; j < TC; ++j) at_b[j] = A_BYTES + turned_at(wc + 32 * j, bc);

    v16f acc[TM][TC] = {};
    copy(0);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    for (i64 stage = 0; stage < stages; ++stage) {
        if (stage + 1 < stages) copy(int(stage + 1) & 1);
        const u8 *tile = staged + (int(stage) & 1) * STAGE;
#pragma unroll
        for (int s = 0; s < GRAD_STEP / 16; ++s) {
            v8bf fa[TM], fb[TC];
#pragma unroll
            for (int i = 0; i < TM; ++i)
                fa[i] = DEPTH_ROWS
                            ? transposed(tile + at_a[i] + s * 16 * BM * 2, 4 * BM * 2)
                            : *reinterpret_cast<const v8bf *>(
                                  tile + at_a[i] + ((2 * s + half) ^ (lane & 7)) * 16);
#pragma unroll
            for (int j = 0; j < TC; ++j)
                fb[j] = transposed(tile + at_b[j] + s * 16 * BC * 2, 4 * BC * 2);
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TC; ++j)
                    acc[i][j] =
                        __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i], fb[j], acc[i][j], 0, 0, 0);
        }
        // The copies are not in the compiler's count of outstanding loads.
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
    }
    T *out = static_cast<T *>(a.out);
#pragma unroll
    for (int j = 0; j < TC; ++j) {
        const i64 c = c0 + wc + 32 * j + (lane & 31);
        if (c >= a.cols) continue;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const i64 m = m0 + wm + 32 * i + 8 * (e / 4) + 4 * half + (e & 3);
                if (m < a.rows) out[m * a.cols + c] = T(acc[i][j][e]);
            }
    }
}

// Sums of `rows` values down each column, 64 columns by 4 rows a workgroup; FP32 sums of chunk
// blockIdx.y in partial, or the result itself where there is one chunk.
constexpr i64 SUM_ROWS = 256;

template <typename T, typename U>
__global__ __launch_bounds__(256) void k_mx_column_sums(const T *x, i64 n, i64 o, i64 ldx, i64 chunk,
                                                        U *out) {
    __shared__ float part[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const i64 c = i64(blockIdx.x) * 64 + lane;
    const i64 first = i64(blockIdx.y) * chunk, last = min(first + chunk, n);
    float sum = 0.0f;
    if (c < o)
        for (i64 r = first + wave; r < last; r += 4) sum += float(x[r * ldx + c]);
    part[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && c < o)
        out[i64(blockIdx.y) * o + c] =
            U((part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]));
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// lanes along a row (a power of two from 32 to 256) and the grid over units and rows.
static int row_lanes(i64 units) {
    int lanes = 5;
    while (lanes < 8 && (i64(1) << lanes) < units) ++lanes;
    return lanes;
}

static dim3 row_grid(i64 units, i64 n, int lanes) {
    const i64 rows = 256 >> lanes;
    return dim3(unsigned((units + (i64(1) << lanes) - 1) >> lanes),
                unsigned(std::min<i64>((n + rows - 1) / rows, 65535)));
}

constexpr i64 MOST = i64(1) << 30;   // rows and columns of an operand

static bool sizes_ok(i64 n, i64 k) { return n >= 1 && k >= 1 && n < MOST && k < MOST; }

// A tile's offsets into dy and the expanded operand stay in 32 bits.
static bool grad_ok(i64 n, i64 k, i64 o) {
    return n >= 1 && k >= 1 && o >= 1 && n < i64(1) << 28 && o <= i64(1) << 22 && k < i64(1) << 24;
}

static int terms_of(int32_t type) { return type == MF_BF16 ? 1 : type == MF_F16 ? 2 : 3; }

static i64 padded(i64 v) { return (v + GRAD_STEP - 1) / GRAD_STEP * GRAD_STEP; }

// BF16 gradients whose contraction is whole steps and whose rows are whole pieces are read in place.
static bool terms_in_place(const void *dy, int32_t type, i64 n, i64 o, i64 ldy, bool depth_rows) {
    return type == MF_BF16 && (depth_rows ? n : o) % GRAD_STEP == 0 && o % 8 == 0 && ldy % 8 == 0 &&
           ldy <= i64(1) << 22 && aligned(dy, 16);
}

static i64 terms_bytes(int32_t type, i64 n, i64 o) {
    return terms_of(type) * padded(n) * padded(o) * 2;
}

// dy's terms: in place, or written to the workspace.
static int make_terms(const void *dy, int32_t type, i64 n, i64 o, i64 ldy, bool depth_rows,
                      void *workspace, i64 bytes, hipStream_t s, GradArgs &args) {
    if (terms_in_place(dy, type, n, o, ldy, depth_rows)) {
        args.a = static_cast<const bf16 *>(dy);
        args.lda = ldy;
        args.width = o;
        args.plane = 0;
        args.terms = 1;
        return MF_OK;
    }
    if (!workspace || bytes < terms_bytes(type, n, o) || !aligned(workspace, 16))
        return fail(MF_E_INVALID, "gradient workspace is missing, unaligned or too small");
    const i64 rows = padded(n), cols = padded(o);
    args.a = static_cast<const bf16 *>(workspace);
    args.lda = args.width = cols;
    args.plane = rows * cols;
    args.terms = terms_of(type);
    const dim3 grid(unsigned((cols + 255) / 256), unsigned(std::min<i64>(rows, 65535)));
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        hipLaunchKernelGGL(k_mx_terms<T>, grid, dim3(256), 0, s, static_cast<const T *>(dy), n, o,
                           ldy, args.terms, rows, cols, static_cast<bf16 *>(workspace));
        return check_launch("gradient terms");
    });
}

static i64 expanded_bytes(i64 depth, i64 k) { return padded(depth) * segments(k) * SEG * 2; }

// dy's terms and the expanded operand, one behind the other.
static i64 grad_bytes(int32_t type, i64 n, i64 o, i64 depth, i64 k) {
    return terms_bytes(type, n, o) + expanded_bytes(depth, k);
}

template <typename T, bool DEPTH_ROWS, int WM, int WC, int TM, int TC>
static int launch_grad_tile(const GradArgs &args, hipStream_t s) {
    constexpr int BM = 32 * WM * TM, BC = 32 * WC * TC, LDS = 2 * (BM + BC) * GRAD_STEP * 2;
    static_assert(BC <= SEG, "a tile's columns are within the padding of the rows");
    const i64 tiles = (args.rows + BM - 1) / BM * ((args.cols + BC - 1) / BC);
    if (tiles > i64(1) << 30) return fail(MF_E_UNSUPPORTED, "gradient too large");
    auto kernel = k_mx_grad<T, DEPTH_ROWS, WM, WC, TM, TC>;
    if (LDS > 64 << 10) {
        const hipError_t e = hipFuncSetAttribute(
            reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (e != hipSuccess) return fail(MF_E_RESOURCE, "LDS of a gradient: %s", hipGetErrorString(e));
    }
    hipLaunchKernelGGL(kernel, dim3(unsigned(tiles)), dim3(64 * WM * WC), LDS, s, args);
    return check_launch("microscaled gradient");
}

template <bool DEPTH_ROWS>
static int launch_grad(GradArgs args, int32_t type, i64 n, i64 o, const u8 *codes, const u8 *scales,
                       void *workspace, i64 bytes, hipStream_t s) {
    if (!workspace || bytes < grad_bytes(type, n, o, args.depth, args.cols) || !aligned(workspace, 16))
        return fail(MF_E_INVALID, "gradient workspace is missing, unaligned or too small");
    const i64 segs = segments(args.cols), rows = padded(args.depth);
    bf16 *const b = reinterpret_cast<bf16 *>(static_cast<u8 *>(workspace) + terms_bytes(type, n, o));
    const dim3 grid(unsigned((segs * 32 + 255) / 256), unsigned(std::min<i64>(rows, 65535)));
    hipLaunchKernelGGL(k_mx_expand, grid, dim3(256), 0, s, reinterpret_cast<const u32 *>(codes), scales,
                       args.depth, segs, DEPTH_ROWS, rows, b);
    args.b = b;
    args.ldb = segs * SEG;
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        // The largest tile of which every compute unit gets one (us, 64 x 64 / 128 x 128 /
        // 256 x 256, n x k x o): dw of 2048 x 11008 x 4096 402 / 262 / 191, dx of it 359 / 277 / 220, dx of
        // 2048 x 4096 x 11008 341 / 200 / 273, dx of 512 x 1024 x 1024 9 / 15 / 31.
        const auto tiles = [&](i64 edge) {
            return (args.rows + edge - 1) / edge * ((args.cols + edge - 1) / edge);
        };
        if (tiles(256) >= 256) return launch_grad_tile<T, DEPTH_ROWS, 2, 4, 4, 2>(args, s);
        if (tiles(128) >= 256) return launch_grad_tile<T, DEPTH_ROWS, 2, 2, 2, 2>(args, s);
        return launch_grad_tile<T, DEPTH_ROWS, 2, 2, 1, 1>(args, s);
    });
}

static int launch_quantize(const void *x, int32_t type, i64 n, i64 k, i64 ldx, bool turned, u8 *codes,
                           u8 *scales, hipStream_t s) {
    if (!x || !codes || !scales || !known_type(type) || !sizes_ok(n, k) || (n > 1 && ldx < k) ||
        !aligned(codes, 16) || !aligned(scales, 8))
        return fail(MF_E_INVALID, "invalid microscaled quantization arguments");
    const i64 units = segments(k) * 32;
    const int lanes = row_lanes(units);
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        const bool vec = aligned(x, 16) && (n == 1 || ldx % PIECE<T> == 0);
        hipLaunchKernelGGL(k_mx_quantize<T>, row_grid(units, n, lanes), dim3(256), 0, s,
                           static_cast<const T *>(x), n, k, ldx, vec, lanes, turned, codes, scales);
        return check_launch("microscaled quantization");
    });
}

// Rows and columns whose scale offsets stay in 32 bits, and depths whose tiles' code offsets do.
static bool product_ok(i64 n, i64 k, i64 o) {
    return n >= 1 && k >= 1 && o >= 1 && n < i64(1) << 28 && o < i64(1) << 28 && k < i64(1) << 24;
}

struct ProductPlan {
    bool few;        // k_mx_few, else k_mx_tile
    bool quantize;   // Q(x) goes through memory
};

constexpr i64 FEW_ROWS = 64;
constexpr i64 FEW_QUANTIZE = 32768;   // values of x that every workgroup may quantize again

static ProductPlan plan_product(i64 n, i64 k, bool keep) {
    const bool few = n <= FEW_ROWS;
    return {few, keep || !few || n > 16 || n * segments(k) * SEG > FEW_QUANTIZE};
}

template <typename T> static int launch_few(const MxArgs &args, const ProductPlan &plan, hipStream_t s) {
    const dim3 grid(unsigned((args.o + FEW_TILE - 1) / FEW_TILE)), block(64 * FEW_WAVES);
    if (!plan.quantize)
        hipLaunchKernelGGL((k_mx_few<T, 1, true>), grid, block, few_lds(args.n, args.segs), s, args);
    else if (args.n <= 16)
        hipLaunchKernelGGL((k_mx_few<T, 1, false>), grid, block, 0, s, args);
    else if (args.n <= 32)
        hipLaunchKernelGGL((k_mx_few<T, 2, false>), grid, block, 0, s, args);
    else if (args.n <= 48)
        hipLaunchKernelGGL((k_mx_few<T, 3, false>), grid, block, 0, s, args);
    else
        hipLaunchKernelGGL((k_mx_few<T, 4, false>), grid, block, 0, s, args);
    return check_launch("microscaled product");
}

template <typename T, int WN, int WO, int TN, int TO>
static int launch_tile(const MxArgs &args, hipStream_t s) {
    constexpr int BN = 32 * WN * TN, BO = 32 * WO * TO, LDS = 2 * (BN + BO) * SEG_BYTES;
    const i64 tiles = (args.n + BN - 1) / BN * ((args.o + BO - 1) / BO);
    if (tiles > i64(1) << 30) return fail(MF_E_UNSUPPORTED, "product too large");
    auto kernel = k_mx_tile<T, WN, WO, TN, TO>;
    if (LDS > 64 << 10) {
        const hipError_t e = hipFuncSetAttribute(
            reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (e != hipSuccess) return fail(MF_E_RESOURCE, "LDS of a product: %s", hipGetErrorString(e));
    }
    hipLaunchKernelGGL(kernel, dim3(unsigned(tiles)), dim3(64 * WN * WO), LDS, s, args);
    return check_launch("microscaled product");
}

template <typename T> static int launch_tiles(const MxArgs &args, hipStream_t s) {
    // The largest tile of which every compute unit gets one (us, 64 x 64 / 128 x 128 / 128 x 256):
    // 2048 x 11008 x 4096 97 / 64 / 62, 2048 x 4096 x 11008 101 / 82 / 77, 300 x 4096 x 4096
    // 12.6 / 18 / 23, 777 x 1500 x 1111 6.1 / 9.5 / 11.8.
    const auto tiles = [&](i64 bn, i64 bo) { return (args.n + bn - 1) / bn * ((args.o + bo - 1) / bo); };
    if (tiles(128, 256) >= 256) return launch_tile<T, 2, 4, 2, 2>(args, s);
    if (tiles(128, 128) >= 256) return launch_tile<T, 2, 2, 2, 2>(args, s);
    return launch_tile<T, 2, 2, 1, 1>(args, s);
}

}  // namespace mf

using namespace mf;

extern "C" {

int mf_mx_quantize(const void *x, int32_t type, int64_t n, int64_t k, int64_t ldx, uint8_t *codes,
                   uint8_t *scales, void *stream) {
    return launch_quantize(x, type, n, k, ldx, false, codes, scales, static_cast<hipStream_t>(stream));
}

int mf_mx_dequantize(const uint8_t *codes, const uint8_t *scales, int64_t n, int64_t k, void *out,
                     int32_t type, void *stream) {
    if (!codes || !scales || !out || !known_type(type) || !sizes_ok(n, k) || !aligned(codes, 16) ||
        !aligned(scales, 8))
        return fail(MF_E_INVALID, "invalid microscaled dequantization arguments");
    const i64 units = (k + 7) / 8;
    const int lanes = row_lanes(units);
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        const bool vec = aligned(out, 16) && (n == 1 || k % PIECE<T> == 0);
        hipLaunchKernelGGL(k_mx_dequantize<T>, row_grid(units, n, lanes), dim3(256), 0,
                           static_cast<hipStream_t>(stream), codes, scales, n, k, vec, lanes,
                           static_cast<T *>(out));
        return check_launch("microscaled dequantization");
    });
}

int mf_mx_linear_sizes(int32_t type, int64_t n, int64_t k, int64_t o, int32_t keep, int64_t *codes,
                       int64_t *workspace) {
    if (!codes || !workspace || !known_type(type) || !product_ok(n, k, o))
        return fail(MF_E_INVALID, "invalid microscaled product sizes");
    const ProductPlan plan = plan_product(n, k, keep);
    *codes = plan.quantize ? n * segments(k) * SEG_BYTES : 0;
    *workspace = plan.few ? 0 : o * segments(k) * SEG_SCALES;
    return MF_OK;
}

int mf_mx_linear(const void *x, int32_t type, int64_t n, int64_t k, int64_t ldx,
                 const uint8_t *wcodes, const uint8_t *wscales, int64_t o, const void *bias,
                 int32_t keep, uint8_t *xcodes, uint8_t *xscales, void *out, void *workspace,
                 int64_t bytes, void *stream) {
    if (!x || !known_type(type) || !product_ok(n, k, o) || (n > 1 && ldx < k) || !wcodes || !wscales ||
        !out || !aligned(wcodes, 16) || !aligned(wscales, 8))
        return fail(MF_E_INVALID, "invalid microscaled product arguments");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const ProductPlan plan = plan_product(n, k, keep);
    if (plan.quantize) {
        const int status = launch_quantize(x, type, n, k, ldx, true, xcodes, xscales, s);
        if (status) return status;
    }
    MxArgs args{};
    args.xc = xcodes;
    args.xs = xscales;
    args.wc = wcodes;
    args.ws = wscales;
    args.x = x;
    args.ldx = ldx;
    args.k = k;
    args.bias = bias;
    args.out = out;
    args.n = n;
    args.o = o;
    args.segs = segments(k);
    if (!plan.few) {
        if (!workspace || bytes < o * args.segs * SEG_SCALES || !aligned(workspace, 8))
            return fail(MF_E_INVALID, "product workspace is missing, unaligned or too small");
        hipLaunchKernelGGL(k_mx_turn_scales, dim3(unsigned((o + 255) / 256), unsigned(args.segs)),
                           dim3(256), 0, s, reinterpret_cast<const v2u *>(wscales), o, args.segs,
                           static_cast<v2u *>(workspace));
        args.ws = static_cast<const u8 *>(workspace);
    }
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        args.vec = aligned(x, 16) && (n == 1 || ldx % PIECE<T> == 0);
        return plan.few ? launch_few<T>(args, plan, s) : launch_tiles<T>(args, s);
    });
}

int mf_mx_grad_workspace(int32_t type, int64_t n, int64_t k, int64_t o, int64_t *bytes) {
    if (!bytes || !known_type(type) || !grad_ok(n, k, o))
        return fail(MF_E_INVALID, "invalid gradient workspace arguments");
    const i64 sums = (n + SUM_ROWS - 1) / SUM_ROWS * o * 4;
    *bytes = std::max(grad_bytes(type, n, o, std::max(n, o), k), sums);
    return MF_OK;
}

int mf_mx_grad_input(const void *dy, int32_t type, int64_t n, int64_t o, int64_t ldy,
                     const uint8_t *wcodes, const uint8_t *wscales, int64_t k, void *dx,
                     void *workspace, int64_t bytes, void *stream) {
    if (!dy || !wcodes || !wscales || !dx || !known_type(type) || !grad_ok(n, k, o) ||
        (n > 1 && ldy < o) || !aligned(wcodes, 16) || !aligned(wscales, 8))
        return fail(MF_E_INVALID, "invalid input gradient arguments");
    hipStream_t s = static_cast<hipStream_t>(stream);
    GradArgs args{};
    const int status = make_terms(dy, type, n, o, ldy, false, workspace, bytes, s, args);
    if (status) return status;
    args.rows = n;
    args.cols = k;
    args.depth = o;
    args.out = dx;
    return launch_grad<false>(args, type, n, o, wcodes, wscales, workspace, bytes, s);
}

int mf_mx_grad_weight(const void *dy, int32_t type, int64_t n, int64_t o, int64_t ldy,
                      const uint8_t *xcodes, const uint8_t *xscales, int64_t k, void *dw,
                      void *workspace, int64_t bytes, void *stream) {
    if (!dy || !xcodes || !xscales || !dw || !known_type(type) || !grad_ok(n, k, o) ||
        (n > 1 && ldy < o) || !aligned(xcodes, 16) || !aligned(xscales, 8))
        return fail(MF_E_INVALID, "invalid weight gradient arguments");
    hipStream_t s = static_cast<hipStream_t>(stream);
    GradArgs args{};
    const int status = make_terms(dy, type, n, o, ldy, true, workspace, bytes, s, args);
    if (status) return status;
    args.rows = o;
    args.cols = k;
    args.depth = n;
    args.out = dw;
    return launch_grad<true>(args, type, n, o, xcodes, xscales, workspace, bytes, s);
}

int mf_mx_grad_bias(const void *dy, int32_t type, int64_t n, int64_t o, int64_t ldy, void *db,
                    void *workspace, int64_t bytes, void *stream) {
    if (!dy || !db || !known_type(type) || !sizes_ok(n, o) || (n > 1 && ldy < o))
        return fail(MF_E_INVALID, "invalid bias gradient arguments");
    hipStream_t s = static_cast<hipStream_t>(stream);
    i64 chunks = (n + SUM_ROWS - 1) / SUM_ROWS;
    if (chunks > 65535) return fail(MF_E_UNSUPPORTED, "too many rows of a bias gradient");
    const unsigned gx = unsigned((o + 63) / 64);
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        const T *x = static_cast<const T *>(dy);
        if (chunks == 1) {
            hipLaunchKernelGGL((k_mx_column_sums<T, T>), dim3(gx), dim3(256), 0, s, x, n, o, ldy, n,
                               static_cast<T *>(db));
            return check_launch("bias gradient");
        }
        if (!workspace || bytes < chunks * o * 4 || !aligned(workspace, 4))
            return fail(MF_E_INVALID, "bias gradient workspace is missing or too small");
        float *part = static_cast<float *>(workspace);
        hipLaunchKernelGGL((k_mx_column_sums<T, float>), dim3(gx, unsigned(chunks)), dim3(256), 0, s,
                           x, n, o, ldy, SUM_ROWS, part);
        hipLaunchKernelGGL((k_mx_column_sums<float, T>), dim3(gx), dim3(256), 0, s, part, chunks, o,
                           o, chunks, static_cast<T *>(db));
        return check_launch("bias gradient");
    });
}

}  // extern "C"
