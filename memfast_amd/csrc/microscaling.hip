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
// row, the others take further rows.
template <typename T>
__global__ __launch_bounds__(256) void k_mx_quantize(const T *x, i64 n, i64 k, i64 ldx, bool vec,
                                                     int lanes, u8 *codes, u8 *scales) {
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
        if ((unit & 3) == 0) scales[r * segs * SEG_SCALES + unit / 4] = u8(byte);
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
    const u8 *xc, *xs;      // [n, segs * 128], [n, segs * 8]
    const u8 *wc, *ws;      // [o, ...]
    const void *bias;       // [o] or nullptr
    void *out;              // [n, o]
    i64 n, o, segs;
};

// A wave takes 32 rows by 32 columns of y straight from global memory.
template <typename T>
__global__ __launch_bounds__(256) void k_mx_mm(const MxArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int half = lane >> 5;
    const i64 n0 = (i64(blockIdx.y) * 2 + (wave >> 1)) * 32;
    const i64 o0 = (i64(blockIdx.x) * 2 + (wave & 1)) * 32;
    if (n0 >= a.n || o0 >= a.o) return;
    // Rows past the end read the last row; their results are not stored.
    const i64 row = min(n0 + (lane & 31), a.n - 1), col = min(o0 + (lane & 31), a.o - 1);
    const u8 *xc = a.xc + row * a.segs * SEG_BYTES + half * 16;
    const u8 *wc = a.wc + col * a.segs * SEG_BYTES + half * 16;
    const u8 *xs = a.xs + row * a.segs * SEG_SCALES, *ws = a.ws + col * a.segs * SEG_SCALES;
    v16f acc = {};
    for (i64 s = 0; s < a.segs; ++s) {
        const u32 sx = half_scales(reinterpret_cast<const v2u *>(xs)[s], half);
        const u32 sw = half_scales(reinterpret_cast<const v2u *>(ws)[s], half);
        const v4u *x4 = reinterpret_cast<const v4u *>(xc + s * SEG_BYTES);
        const v4u *w4 = reinterpret_cast<const v4u *>(wc + s * SEG_BYTES);
        acc = mfma_step<0>(x4[0], w4[0], acc, sx, sw);
        acc = mfma_step<1>(x4[2], w4[2], acc, sx, sw);
        acc = mfma_step<2>(x4[4], w4[4], acc, sx, sw);
        acc = mfma_step<3>(x4[6], w4[6], acc, sx, sw);
    }
    const i64 c = o0 + (lane & 31);
    if (c >= a.o) return;
    const float bias = a.bias ? float(static_cast<const T *>(a.bias)[c]) : 0.0f;
    T *out = static_cast<T *>(a.out);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const i64 r = n0 + 8 * (i / 4) + 4 * half + (i & 3);
        if (r < a.n) out[r * a.o + c] = T(acc[i] + bias);
    }
}

// ---------------------------------------------------------------------------
// Gradients
// ---------------------------------------------------------------------------
constexpr int GRAD_TILE = 128, GRAD_STEP = 64;
constexpr int GRAD_PITCH = 160;   // BF16 values of an LDS row of 128, padded against bank conflicts

struct GradArgs {
    const bf16 *a;          // dy terms: plane t at a + t * plane, rows of lda values
    i64 plane, lda;
    i64 width;              // values of a row that may be read, a multiple of 8
    int terms;
    const u8 *codes, *scales;   // the 4-bit operand [contraction, segs * 128]
    i64 segs;
    i64 rows, cols;         // of the result
    i64 depth;              // contraction
    void *out;              // [rows, cols]
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

typedef __attribute__((address_space(3))) v4s *lds_v4s;

// Four rows by sixteen columns per sixteen lanes, transposed: the lane gets its column's values
// of rows c .. c + 3 (and, with a second read, c + 4 .. c + 7).
__device__ __forceinline__ v8bf transposed(const bf16 *tile, int c, int col, int lane) {
    const int i = lane & 15;
    const bf16 *p = tile + (c + (i >> 2)) * GRAD_PITCH + col + 4 * (i & 3);
    union {
        v4s s[2];
        v8bf v;
    } u;
    u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(p));
    u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(p + 4 * GRAD_PITCH));
    return u.v;
}

// The 32 values of a block as BF16.
__device__ __forceinline__ void expand_block(v4u codes, u32 byte, bf16 *to) {
    const float scale = scale_of(byte);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        float v[8];
        values8(codes[w], scale, v);
        v8bf out;
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = bf16(v[i]);
        *reinterpret_cast<v8bf *>(to + 8 * w) = out;
    }
}

// out[m, c] = sum_t sum_d A_t[m, d] B[d, c] over 128 x 128 tiles, 64 of the contraction at a time.
// DEPTH_ROWS: A's rows run along the contraction (dw: A is dy^T); else along m (dx).
// A has GRAD_STEP-padded contraction with zeros in the padding, B's rows past depth are zeros here.
template <typename T, bool DEPTH_ROWS>
__global__ __launch_bounds__(256) void k_mx_grad(const GradArgs a) {
    __shared__ alignas(16) bf16 tile_a[GRAD_TILE * GRAD_STEP > GRAD_STEP * GRAD_PITCH ? GRAD_TILE * GRAD_STEP
                                                                         : GRAD_STEP * GRAD_PITCH];
    __shared__ alignas(16) bf16 tile_b[GRAD_STEP * GRAD_PITCH];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const i64 m0 = i64(blockIdx.y) * GRAD_TILE, c0 = i64(blockIdx.x) * GRAD_TILE;
    const int wm = (wave >> 1) * 64, wc = (wave & 1) * 64;
    const int tr_col = 16 * ((lane >> 4) & 1), tr_row = 8 * (lane >> 5);
    v16f acc[2][2] = {};
    for (int t = a.terms - 1; t >= 0; --t) {
        const bf16 *plane = a.a + t * a.plane;
        for (i64 d0 = 0; d0 < a.depth; d0 += GRAD_STEP) {
            __syncthreads();
            if (DEPTH_ROWS) {   // 64 rows of 128 values, 16 pieces each
                for (int u = tid; u < GRAD_STEP * 16; u += 256) {
                    const int r = u >> 4, p = u & 15;
                    const i64 m = min(m0 + p * 8, a.width - 8);
                    *reinterpret_cast<v4u *>(tile_a + r * GRAD_PITCH + p * 8) =
                        *reinterpret_cast<const v4u *>(plane + (d0 + r) * a.lda + m);
                }
            } else {            // 128 rows of 64 values, 8 pieces each, rotated by the row
                for (int u = tid; u < GRAD_TILE * 8; u += 256) {
                    const int r = u >> 3, p = u & 7;
                    const i64 m = min(m0 + r, a.rows - 1);
                    *reinterpret_cast<v4u *>(tile_a + r * GRAD_STEP + (p ^ (r & 7)) * 8) =
                        *reinterpret_cast<const v4u *>(plane + m * a.lda + d0 + p * 8);
                }
            }
            {                   // 64 rows of four blocks: one block a thread
                const int r = tid >> 2, b = tid & 3;
                const i64 d = d0 + r;
                v4u codes = {0, 0, 0, 0};
                u32 byte = 1;
                if (d < a.depth) {
                    codes = *reinterpret_cast<const v4u *>(a.codes + d * a.segs * SEG_BYTES +
                                                           c0 / 2 + b * 16);
                    byte = a.scales[d * a.segs * SEG_SCALES + c0 / 32 + b];
                }
                expand_block(codes, byte, tile_b + r * GRAD_PITCH + b * 32);
            }
            __syncthreads();
#pragma unroll
            for (int s = 0; s < GRAD_STEP / 16; ++s) {
                v8bf fa[2], fb[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (DEPTH_ROWS) {
                        fa[i] = transposed(tile_a, 16 * s + tr_row, wm + 32 * i + tr_col, lane);
                    } else {
                        const int r = wm + 32 * i + (lane & 31), p = 2 * s + (lane >> 5);
                        fa[i] = *reinterpret_cast<const v8bf *>(tile_a + r * GRAD_STEP +
                                                                (p ^ (r & 7)) * 8);
                    }
                    fb[i] = transposed(tile_b, 16 * s + tr_row, wc + 32 * i + tr_col, lane);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i], fb[j],
                                                                            acc[i][j], 0, 0, 0);
            }
        }
    }
    T *out = static_cast<T *>(a.out);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const i64 c = c0 + wc + 32 * j + (lane & 31);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const i64 m = m0 + wm + 32 * i + 8 * (e / 4) + 4 * (lane >> 5) + (e & 3);
                if (m < a.rows && c < a.cols) out[m * a.cols + c] = T(acc[i][j][e]);
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

static int terms_of(int32_t type) { return type == MF_BF16 ? 1 : type == MF_F16 ? 2 : 3; }

static i64 padded(i64 v) { return (v + GRAD_STEP - 1) / GRAD_STEP * GRAD_STEP; }

// BF16 gradients whose contraction is whole steps and whose rows are whole pieces are read in place.
static bool terms_in_place(const void *dy, int32_t type, i64 n, i64 o, i64 ldy, bool depth_rows) {
    return type == MF_BF16 && (depth_rows ? n : o) % GRAD_STEP == 0 && o % 8 == 0 && ldy % 8 == 0 &&
           aligned(dy, 16);
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

template <bool DEPTH_ROWS> static int launch_grad(const GradArgs &args, int32_t type, hipStream_t s) {
    const i64 gx = (args.cols + GRAD_TILE - 1) / GRAD_TILE, gy = (args.rows + GRAD_TILE - 1) / GRAD_TILE;
    if (gy > 65535) return fail(MF_E_UNSUPPORTED, "too many rows of a gradient");
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        hipLaunchKernelGGL((k_mx_grad<T, DEPTH_ROWS>), dim3(unsigned(gx), unsigned(gy)), dim3(256), 0,
                           s, args);
        return check_launch("microscaled gradient");
    });
}

}  // namespace mf

using namespace mf;

extern "C" {

int mf_mx_quantize(const void *x, int32_t type, int64_t n, int64_t k, int64_t ldx, uint8_t *codes,
                   uint8_t *scales, void *stream) {
    if (!x || !codes || !scales || !known_type(type) || !sizes_ok(n, k) || (n > 1 && ldx < k) ||
        !aligned(codes, 16) || !aligned(scales, 8))
        return fail(MF_E_INVALID, "invalid microscaled quantization arguments");
    const i64 units = segments(k) * 32;
    const int lanes = row_lanes(units);
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        const bool vec = aligned(x, 16) && (n == 1 || ldx % PIECE<T> == 0);
        hipLaunchKernelGGL(k_mx_quantize<T>, row_grid(units, n, lanes), dim3(256), 0,
                           static_cast<hipStream_t>(stream), static_cast<const T *>(x), n, k, ldx,
                           vec, lanes, codes, scales);
        return check_launch("microscaled quantization");
    });
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

int mf_mx_linear(const void *x, int32_t type, int64_t n, int64_t k, int64_t ldx,
                 const uint8_t *wcodes, const uint8_t *wscales, int64_t o, const void *bias,
                 uint8_t *xcodes, uint8_t *xscales, void *out, void *stream) {
    if (!wcodes || !wscales || !out || o < 1 || o >= MOST || !aligned(wcodes, 16) ||
        !aligned(wscales, 8))
        return fail(MF_E_INVALID, "invalid microscaled product arguments");
    const int status = mf_mx_quantize(x, type, n, k, ldx, xcodes, xscales, stream);
    if (status) return status;
    const MxArgs args{xcodes, xscales, wcodes, wscales, bias, out, n, o, segments(k)};
    if ((n + 63) / 64 > 65535) return fail(MF_E_UNSUPPORTED, "too many rows of a product");
    const dim3 grid(unsigned((o + 63) / 64), unsigned((n + 63) / 64));
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        hipLaunchKernelGGL(k_mx_mm<T>, grid, dim3(256), 0, static_cast<hipStream_t>(stream), args);
        return check_launch("microscaled product");
    });
}

int mf_mx_grad_workspace(int32_t type, int64_t n, int64_t o, int64_t *bytes) {
    if (!bytes || !known_type(type) || !sizes_ok(n, o))
        return fail(MF_E_INVALID, "invalid gradient workspace arguments");
    const i64 sums = (n + SUM_ROWS - 1) / SUM_ROWS * o * 4;
    *bytes = std::max(terms_bytes(type, n, o), sums);
    return MF_OK;
}

int mf_mx_grad_input(const void *dy, int32_t type, int64_t n, int64_t o, int64_t ldy,
                     const uint8_t *wcodes, const uint8_t *wscales, int64_t k, void *dx,
                     void *workspace, int64_t bytes, void *stream) {
    if (!dy || !wcodes || !wscales || !dx || !known_type(type) || !sizes_ok(n, o) || !sizes_ok(n, k) ||
        (n > 1 && ldy < o) || !aligned(wcodes, 16) || !aligned(wscales, 8))
        return fail(MF_E_INVALID, "invalid input gradient arguments");
    hipStream_t s = static_cast<hipStream_t>(stream);
    GradArgs args{};
    const int status = make_terms(dy, type, n, o, ldy, false, workspace, bytes, s, args);
    if (status) return status;
    args.codes = wcodes;
    args.scales = wscales;
    args.segs = segments(k);
    args.rows = n;
    args.cols = k;
    args.depth = o;
    args.out = dx;
    return launch_grad<false>(args, type, s);
}

int mf_mx_grad_weight(const void *dy, int32_t type, int64_t n, int64_t o, int64_t ldy,
                      const uint8_t *xcodes, const uint8_t *xscales, int64_t k, void *dw,
                      void *workspace, int64_t bytes, void *stream) {
    if (!dy || !xcodes || !xscales || !dw || !known_type(type) || !sizes_ok(n, o) || !sizes_ok(n, k) ||
        (n > 1 && ldy < o) || !aligned(xcodes, 16) || !aligned(xscales, 8))
        return fail(MF_E_INVALID, "invalid weight gradient arguments");
    hipStream_t s = static_cast<hipStream_t>(stream);
    GradArgs args{};
    const int status = make_terms(dy, type, n, o, ldy, true, workspace, bytes, s, args);
    if (status) return status;
    args.codes = xcodes;
    args.scales = xscales;
    args.segs = segments(k);
    args.rows = o;
    args.cols = k;
    args.depth = n;
    args.out = dw;
    return launch_grad<true>(args, type, s);
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
