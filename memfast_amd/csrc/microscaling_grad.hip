// Gradients of the product of two 4-bit operands, straight through the quantizers:
//   dx = dy Q(W), dw = dy^T Q(x), db = sum_n dy.
// They contract over the rows of the 4-bit operand, whose scales change from row to row, so the block
// scales of the matrix instruction cannot carry them. A code times its scale is exact in BF16 (two
// significant bits), so the 4-bit operand is expanded to BF16 once, and dy enters as BF16 terms whose
// sum is its value exactly: one for BF16, two for FP16, three for FP32. The products of the
// terms are exact, and the sums FP32.
#include <algorithm>
#include <type_traits>

#include "mf_mx.h"

namespace mf {

constexpr int GRAD_STEP = 64;     // of the contraction in one stage
constexpr i64 SUM_ROWS = 256;     // rows of dy in one partial sum

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

struct ExpandJob {
    Job job;
    const u32 *codes;   // [n, segs * 32]
    Scales scales;
    i64 n, rows;        // zeros from row n to rows
    bf16 *out;          // [rows, segs * 256]
};

// What the products read, in one launch: dy's terms, both operands in BF16, and dy's column sums.
struct PrepareArgs {
    const void *dy;     // [n, o], rows ldy apart
    i64 n, o, ldy;
    bool vec;
    Job terms;
    int term_count;
    i64 rows, cols;     // n and o in whole steps
    bf16 *planes;       // [term_count][rows][cols], zeros past n and o
    ExpandJob expand[2];
    i64 segs;
    Job sums;           // blocks of 64 columns and SUM_ROWS rows
    float *partial;     // [gy, o], or the result
    void *db;           // with one block of rows
};

// dy's terms add up to its value exactly (each takes eight significant bits by truncation, which also
// keeps the largest finite values finite). A lane takes eight values.
template <typename T> __device__ __forceinline__ void write_terms(const PrepareArgs &a) {
    const i64 unit = a.terms.unit();
    if (unit * 8 >= a.cols) return;
    for (i64 r = a.terms.row(); r < a.rows; r += a.terms.step()) {
        float rest[8] = {};
        if (r < a.n) load8(static_cast<const T *>(a.dy) + r * a.ldy, unit * 8, a.o, a.vec, rest);
        for (int t = 0; t < a.term_count; ++t) {
            v8bf out;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const u32 bits = __float_as_uint(rest[i]);
                if ((bits & 0x7f800000u) == 0x7f800000u) {  // a NaN or an infinity is one term
                    out[i] = bf16(rest[i]);
                    rest[i] = 0.0f;
                } else {
                    const float term = __uint_as_float(bits & 0xffff0000u);
                    out[i] = bf16(term);
                    rest[i] -= term;
                }
            }
            *reinterpret_cast<v8bf *>(a.planes + (t * a.rows + r) * a.cols + unit * 8) = out;
        }
    }
}

__device__ __forceinline__ void expand_rows(const ExpandJob &e, i64 segs) {
    const i64 unit = e.job.unit();
    if (unit >= segs * 32) return;
    for (i64 r = e.job.row(); r < e.rows; r += e.job.step()) {
        v8bf v = {};
        if (r < e.n)
            v = expand8(e.codes[r * segs * 32 + unit],
                        e.scales.data[r * e.scales.row + unit / 32 * e.scales.seg + (unit / 4 & 7)]);
        *reinterpret_cast<v8bf *>(e.out + (r * segs * 32 + unit) * 8) = v;
    }
}

// Column sums of a block of rows in FP32, four rows at a time.
template <typename T, typename U>
__device__ __forceinline__ void column_sums(const T *x, i64 o, i64 ldx, i64 first, i64 last, i64 c,
                                            float (&part)[4][64], U *out) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float sum = 0.0f;
    if (c < o)
        for (i64 r = first + wave; r < last; r += 4) sum += float(x[r * ldx + c]);
    part[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && c < o)
        out[c] = U((part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]));
}

// Bound by its bytes: for 2048 x 11008 x 4096 BF16, where dy is read in place, 170 MB in 33 us, 5.1 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void k_mx_prepare(const PrepareArgs a) {
    __shared__ float part[4][64];
    if (a.terms.mine(blockIdx.x)) {
        write_terms<T>(a);
    } else if (a.sums.mine(blockIdx.x)) {
        const i64 chunk = (blockIdx.x - a.sums.first) / a.sums.gx, c = a.sums.unit();
        const i64 first = chunk * SUM_ROWS, last = min(first + SUM_ROWS, a.n);
        const T *dy = static_cast<const T *>(a.dy);
        if (a.sums.gy == 1)
            column_sums(dy, a.o, a.ldy, first, last, c, part, static_cast<T *>(a.db));
        else
            column_sums(dy, a.o, a.ldy, first, last, c, part, a.partial + chunk * a.o);
    } else {
        expand_rows(a.expand[a.expand[1].job.mine(blockIdx.x) ? 1 : 0], a.segs);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void k_mx_sum_partials(const float *partial, i64 chunks, i64 o, T *db) {
    __shared__ float part[4][64];
    column_sums(partial, o, o, 0, chunks, i64(blockIdx.x) * 64 + (threadIdx.x & 63), part, db);
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

// Where piece p of row r of a tile with that many pieces a row lies in LDS, and the piece that lies at p:
// moved on so that four consecutive rows' reads of 64 bytes are in different banks (rows of 384
// bytes are half a turn of the banks apart from each other already).
template <int PIECES> __device__ __forceinline__ int moved(int p, int r) {
    static_assert(PIECES == 8 || PIECES == 16 || PIECES == 24 || PIECES == 32, "widths of tiles");
    return (p + (PIECES == 8 ? 4 * (r >> 1 & 1) : 4 * (r & 3))) % PIECES;
}
template <int PIECES> __device__ __forceinline__ int moved_back(int p, int r) {
    return (p + PIECES - (PIECES == 8 ? 4 * (r >> 1 & 1) : 4 * (r & 3))) % PIECES;
}

// Tile `block` of out[m, c] = sum_t sum_d A_t[m, d] B[d, c], WM x WC waves of TM x TC tiles of 32 x 32,
// 64 of the contraction a stage, copied to LDS without passing through registers, STAGES - 1 stages
// ahead of the matrix cores.
// DEPTH_ROWS: A's rows run along the contraction (dw: A is dy^T); else along m (dx). Operands whose rows
// run along the contraction are read transposed, four rows of 16 columns by 16 lanes.
// Bound by the matrix cores: dx of 4096^3 with one term 116 us, 1185 TFLOP/s, a BF16 product's rate; dx and dw
// of 2048 x 11008 x 4096, each repeated alone with its expansion, 188 and 187 us, 980 TFLOP/s, with a last
// round of tiles that fills part of the chip. Between the other kernels of a training step the profiler
// shows a tenth more for the kernels alone. Two and three terms: dx of it 342 and 516 us, dw 329 and 503.
template <typename T, bool DEPTH_ROWS, int WM, int WC, int TM, int TC, int STAGES>
__device__ __forceinline__ void grad_tile(const GradArgs &a, u32 block, u8 *staged) {
    constexpr int BM = 32 * WM * TM, BC = 32 * WC * TC, WAVES = WM * WC;
    constexpr int A_BYTES = BM * GRAD_STEP * 2, STAGE = (BM + BC) * GRAD_STEP * 2;
    constexpr int COPIES = STAGE / 1024 / WAVES;
    static_assert(STAGE % (1024 * WAVES) == 0 && A_BYTES % 1024 == 0, "whole copies");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    u32 tx, ty;
    xcd_tile(block, u32((a.rows + BM - 1) / BM), u32((a.cols + BC - 1) / BC), tx, ty);
    const i64 m0 = i64(tx) * BM, c0 = i64(ty) * BC;

    const int first_copy = __builtin_amdgcn_readfirstlane(wave * COPIES);
    u32 offset[COPIES];
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
        const int at = (first_copy + i) * 1024;
        if (at < A_BYTES && !DEPTH_ROWS) {      // rows of 64 values, 8 pieces at p ^ (r / 2 & 7)
            const int piece = at / 16 + lane, r = piece >> 3;
            offset[i] = u32(min(i64(r), a.rows - m0 - 1) * a.lda * 2) + u32(((piece ^ r >> 1) & 7) * 16);
        } else if (at < A_BYTES) {
            constexpr int PIECES = BM / 8;
            const int piece = at / 16 + lane, r = piece / PIECES;
            const int p = moved_back<PIECES>(piece % PIECES, r);
            offset[i] = u32(r * a.lda * 2) + u32(min(m0 + p * 8, a.width - 8) - m0) * 2;
        } else {
            constexpr int PIECES = BC / 8;
            const int piece = (at - A_BYTES) / 16 + lane, r = piece / PIECES;
            const int p = moved_back<PIECES>(piece % PIECES, r);
            offset[i] = u32(r * a.ldb * 2) + u32(min(c0 + p * 8, a.ldb - 8) - c0) * 2;
        }
    }
    const u32 lds = lds_address(staged);
    const i64 steps = (a.depth + GRAD_STEP - 1) / GRAD_STEP, stages = steps * a.terms;
    // The next copy's tiles; the smallest terms come first.
    const i64 a_step = (DEPTH_ROWS ? GRAD_STEP * a.lda : GRAD_STEP) * 2, b_step = GRAD_STEP * a.ldb * 2;
    const u8 *at_a0 = reinterpret_cast<const u8 *>(a.a + (a.terms - 1) * a.plane +
                                                   (DEPTH_ROWS ? m0 : m0 * a.lda));
    const u8 *at_b0 = reinterpret_cast<const u8 *>(a.b + c0);
    i64 step = 0;
    auto copy = [&](int buffer) {
#pragma unroll
        for (int i = 0; i < COPIES; ++i) {
            const int at = (first_copy + i) * 1024;
            lds_dma_16((at < A_BYTES ? at_a0 : at_b0) + offset[i],
                       __builtin_amdgcn_readfirstlane(lds + buffer * STAGE + at));
        }
        at_a0 += a_step;
        at_b0 += b_step;
        if (++step == steps) {
            step = 0;
            at_a0 -= steps * a_step + a.plane * 2;
            at_b0 -= steps * b_step;
        }
    };

    // Where this lane's fragments start in a stage.
    const int wm = (wave / WC) * TM * 32, wc = (wave % WC) * TC * 32;
    const int i16 = lane & 15, side = lane >> 4 & 1, half = lane >> 5;
    int at_a[TM], at_b[TC];
    auto turned_at = [&](int col, auto width) {
        constexpr int PIECES = decltype(width)::value / 8;
        const int r = 8 * half + (i16 >> 2), piece = (col + 16 * side) / 8 + (i16 & 3) / 2;
        return r * PIECES * 16 + moved<PIECES>(piece, r) * 16 + (i16 & 1) * 8;
    };
    const std::integral_constant<int, BM> bm{};
    const std::integral_constant<int, BC> bc{};
#pragma unroll
    for (int i = 0; i < TM; ++i)
        at_a[i] = DEPTH_ROWS ? turned_at(wm + 32 * i, bm) : (wm + 32 * i + (lane & 31)) * GRAD_STEP * 2;
#pragma unroll
    for (int j = 0; j < TC; ++j) at_b[j] = A_BYTES + turned_at(wc + 32 * j, bc);

    v16f acc[TM][TC] = {};
    int filling = 0, reading = 0;
    i64 next = 0;
    for (; next < STAGES - 1 && next < stages; ++next) copy(filling++);
    for (i64 stage = 0; stage < stages; ++stage) {
        // All copies but those of the STAGES - 2 stages behind this one have to be there; near the
        // end there are fewer behind.
        if (stage + STAGES - 2 < stages)
            wait_stage<(STAGES - 2) * COPIES>();
        else
            wait_stage<0>();
        const u8 *tile = staged + reading * STAGE;
        reading = reading + 1 == STAGES ? 0 : reading + 1;
        auto multiply = [&](int s) {
            v8bf fa[TM], fb[TC];
#pragma unroll
            for (int i = 0; i < TM; ++i)
                fa[i] = DEPTH_ROWS
                            ? transposed(tile + at_a[i] + s * 16 * BM * 2, 4 * BM * 2)
                            : *reinterpret_cast<const v8bf *>(
                                  tile + at_a[i] + ((2 * s + half) ^ (lane >> 1 & 7)) * 16);
#pragma unroll
            for (int j = 0; j < TC; ++j)
                fb[j] = transposed(tile + at_b[j] + s * 16 * BC * 2, 4 * BC * 2);
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TC; ++j)
                    acc[i][j] =
                        __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i], fb[j], acc[i][j], 0, 0, 0);
        };
        if (next < stages) {
            copy(filling);
            ++next;
            filling = filling + 1 == STAGES ? 0 : filling + 1;
        }
#pragma unroll
        for (int s = 0; s < GRAD_STEP / 16; ++s) multiply(s);
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

template <typename T, bool DEPTH_ROWS, int WM, int WC, int TM, int TC, int STAGES>
__global__ __launch_bounds__(64 * WM * WC) void k_mx_grad(const GradArgs a) {
    extern __shared__ __align__(16) u8 staged[];
    grad_tile<T, DEPTH_ROWS, WM, WC, TM, TC, STAGES>(a, blockIdx.x, staged);
}

// Both products in one launch, where neither fills the chip.
template <typename T, int WM, int WC, int TM, int TC, int STAGES>
__global__ __launch_bounds__(64 * WM * WC) void k_mx_grads(const GradArgs dx, const GradArgs dw,
                                                           u32 dx_tiles) {
    extern __shared__ __align__(16) u8 staged[];
    if (blockIdx.x < dx_tiles)
        grad_tile<T, false, WM, WC, TM, TC, STAGES>(dx, blockIdx.x, staged);
    else
        grad_tile<T, true, WM, WC, TM, TC, STAGES>(dw, blockIdx.x - dx_tiles, staged);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// A tile's offsets into dy and the expanded operand stay in 32 bits.
static bool grad_ok(i64 n, i64 k, i64 o) {
    return n >= 1 && k >= 1 && o >= 1 && n < i64(1) << 24 && o <= i64(1) << 22 && k < i64(1) << 24;
}

static int terms_of(int32_t type) { return type == MF_BF16 ? 1 : type == MF_F16 ? 2 : 3; }

static i64 padded(i64 v) { return (v + GRAD_STEP - 1) / GRAD_STEP * GRAD_STEP; }

// BF16 gradients whose contraction is whole steps and whose rows are whole pieces are read in place.
static bool in_place(const void *dy, int32_t type, i64 o, i64 ldy, i64 depth) {
    return type == MF_BF16 && depth % GRAD_STEP == 0 && o % 8 == 0 && ldy % 8 == 0 &&
           ldy <= i64(1) << 22 && aligned(dy, 16);
}

struct GradSpace {
    i64 terms, weight, input, sums, bytes;      // where each part begins, and the end
    GradSpace(int32_t type, i64 n, i64 k, i64 o, bool dx, bool dw, bool db) {
        const i64 width = segments(k) * SEG * 2, chunks = (n + SUM_ROWS - 1) / SUM_ROWS;
        terms = 0;
        weight = terms + (dx || dw ? terms_of(type) * padded(n) * padded(o) * 2 : 0);
        input = weight + (dx ? padded(o) * width : 0);
        sums = input + (dw ? padded(n) * width : 0);
        bytes = sums + (db && chunks > 1 ? chunks * o * 4 : 0);
    }
};

static i64 grad_tiles(const GradArgs &a, i64 bm, i64 bc) {
    return (a.rows + bm - 1) / bm * ((a.cols + bc - 1) / bc);
}

template <typename T, bool DEPTH_ROWS, int WM, int WC, int TM, int TC, int STAGES>
static int launch_grad_tile(const GradArgs &args, hipStream_t s) {
    constexpr int BM = 32 * WM * TM, BC = 32 * WC * TC, LDS = STAGES * (BM + BC) * GRAD_STEP * 2;
    const i64 tiles = grad_tiles(args, BM, BC);
    if (tiles > i64(1) << 30) return fail(MF_E_UNSUPPORTED, "gradient too large");
    auto kernel = k_mx_grad<T, DEPTH_ROWS, WM, WC, TM, TC, STAGES>;
    if (const int status = allow_lds(kernel, LDS)) return status;
    hipLaunchKernelGGL(kernel, dim3(unsigned(tiles)), dim3(64 * WM * WC), LDS, s, args);
    return check_launch("microscaled gradient");
}

// The tile whose rounds over the 256 compute units take the least: a round of 256 x 256 takes 117 us
// at a depth of 4096, one of 192 x 256 0.75 and one of 128 x 128 (two a compute unit) 0.65 of that. us,
// 256 x 256 / 192 x 256 / 128 x 128, n x k x o: dx of 2048 x 11008 x 4096 (344 / 473 / 1376 tiles)
// 220 / 187 / 268, dw of it 187 / 206 / 251, dx of 2048 x 4096 x 11008 264 / 220 / 198, dx of 4096^3 116 / 162 / 159.
// Where 128 x 128 leaves compute units without a tile, 64 x 64: dx of 512 x 1024 x 1024 8 against 15 us. Few
// small tiles wait for their copies: a third stage takes dx of 128 x 4096 x 4096 from 34 to 24 us; in
// the larger ones it costs the second workgroup (282 -> 321 us).
template <typename T, bool DEPTH_ROWS> static int launch_grad(const GradArgs &args, hipStream_t s) {
    if (grad_tiles(args, 128, 128) < 256) return launch_grad_tile<T, DEPTH_ROWS, 2, 2, 1, 1, 3>(args, s);
    const auto rounds = [](i64 tiles, i64 at_once) { return (tiles + at_once - 1) / at_once; };
    const i64 large = rounds(grad_tiles(args, 256, 256), 256) * 100;
    const i64 middle = rounds(grad_tiles(args, 192, 256), 256) * 75;
    const i64 small = rounds(grad_tiles(args, 128, 128), 512) * 65;
    if (large <= middle && large <= small) return launch_grad_tile<T, DEPTH_ROWS, 4, 2, 2, 4, 2>(args, s);
    if (middle <= small) return launch_grad_tile<T, DEPTH_ROWS, 2, 4, 3, 2, 2>(args, s);
    return launch_grad_tile<T, DEPTH_ROWS, 2, 2, 2, 2, 2>(args, s);
}

template <typename T> static int launch_both(const GradArgs &dx, const GradArgs &dw, hipStream_t s) {
    const i64 tiles = grad_tiles(dx, 64, 64);
    constexpr int STAGES = 3, LDS = STAGES * 128 * GRAD_STEP * 2;
    if (grad_tiles(dx, 128, 128) < 256 && grad_tiles(dw, 128, 128) < 256) {
        auto kernel = k_mx_grads<T, 2, 2, 1, 1, STAGES>;
        if (const int status = allow_lds(kernel, LDS)) return status;
        hipLaunchKernelGGL(kernel, dim3(unsigned(tiles + grad_tiles(dw, 64, 64))), dim3(256), LDS, s, dx, dw,
                           u32(tiles));
        return check_launch("microscaled gradients");
    }
    const int status = launch_grad<T, false>(dx, s);
    return status ? status : launch_grad<T, true>(dw, s);
}

}  // namespace mf

using namespace mf;

extern "C" {

int mf_mx_grads_workspace(int32_t type, int64_t n, int64_t k, int64_t o, int32_t dx, int32_t dw,
                          int32_t db, int64_t *bytes) {
    if (!bytes || !known_type(type) || !grad_ok(n, k, o))
        return fail(MF_E_INVALID, "invalid gradient workspace arguments");
    *bytes = GradSpace(type, n, k, o, dx, dw, db).bytes;
    return MF_OK;
}

int mf_mx_grads(const void *dy, int32_t type, int64_t n, int64_t o, int64_t ldy,
                const uint8_t *wcodes, const uint8_t *wscales, int32_t by_segment,
                const uint8_t *xcodes, const uint8_t *xscales, int64_t k, void *dx, void *dw, void *db,
                void *workspace, int64_t bytes, void *stream) {
    if (!dy || !known_type(type) || !grad_ok(n, k, o) || (n > 1 && ldy < o) || !(dx || dw || db) ||
        (dx && (!wcodes || !wscales || !aligned(wcodes, 16))) ||
        (dw && (!xcodes || !xscales || !aligned(xcodes, 16))))
        return fail(MF_E_INVALID, "invalid gradient arguments");
    const GradSpace space(type, n, k, o, dx, dw, db);
    if (space.bytes && (!workspace || bytes < space.bytes || !aligned(workspace, 16)))
        return fail(MF_E_INVALID, "gradient workspace is missing, unaligned or too small");
    hipStream_t s = static_cast<hipStream_t>(stream);
    u8 *const base = static_cast<u8 *>(workspace);
    const i64 segs = segments(k), chunks = (n + SUM_ROWS - 1) / SUM_ROWS;
    return with_type(type, [&](auto zero) -> int {
        using T = decltype(zero);
        PrepareArgs p{};
        u32 blocks = 0;
        p.dy = dy;
        p.n = n;
        p.o = o;
        p.ldy = ldy;
        p.vec = aligned(dy, 16) && (n == 1 || ldy % PIECE<T> == 0);
        p.segs = segs;
        // dx contracts over o, dw over n.
        const bool dx_in_place = dx && in_place(dy, type, o, ldy, o);
        const bool dw_in_place = dw && in_place(dy, type, o, ldy, n);
        p.rows = padded(n);
        p.cols = padded(o);
        p.term_count = terms_of(type);
        p.planes = reinterpret_cast<bf16 *>(base + space.terms);
        if ((dx && !dx_in_place) || (dw && !dw_in_place))
            p.terms = add_job(p.cols / 8, p.rows, blocks);
        GradArgs args[2]{};
        for (int i = 0; i < 2; ++i) {
            GradArgs &a = args[i];
            if (i == 0 ? dx_in_place : dw_in_place) {
                a.a = static_cast<const bf16 *>(dy);
                a.lda = ldy;
                a.width = o;
                a.terms = 1;
            } else {
                a.a = p.planes;
                a.lda = a.width = p.cols;
                a.plane = p.rows * p.cols;
                a.terms = p.term_count;
            }
            a.b = reinterpret_cast<bf16 *>(base + (i == 0 ? space.weight : space.input));
            a.ldb = segs * SEG;
            a.cols = k;
            a.rows = i == 0 ? n : o;
            a.depth = i == 0 ? o : n;
            a.out = i == 0 ? dx : dw;
            if (!a.out) continue;
            p.expand[i] = {add_job(segs * 32, padded(a.depth), blocks),
                           reinterpret_cast<const u32 *>(i == 0 ? wcodes : xcodes),
                           i == 1 ? scales_by_segment(xscales, n)
                                  : by_segment ? scales_by_segment(wscales, o) : scales_by_row(wscales, segs),
                           a.depth, padded(a.depth), const_cast<bf16 *>(a.b)};
        }
        if (db) {
            p.sums = {blocks, u32((o + 63) / 64), u32(chunks), 6};
            blocks += p.sums.gx * p.sums.gy;
            p.partial = reinterpret_cast<float *>(base + space.sums);
            p.db = db;
        }
        hipLaunchKernelGGL(k_mx_prepare<T>, dim3(blocks), dim3(256), 0, s, p);
        if (const int status = check_launch("gradient operands")) return status;
        if (db && chunks > 1) {
            hipLaunchKernelGGL(k_mx_sum_partials<T>, dim3(p.sums.gx), dim3(256), 0, s, p.partial, chunks,
                               o, static_cast<T *>(db));
            if (const int status = check_launch("bias gradient")) return status;
        }
        if (dx && dw) return launch_both<T>(args[0], args[1], s);
        if (dx) return launch_grad<T, false>(args[0], s);
        return dw ? launch_grad<T, true>(args[1], s) : int(MF_OK);
    });
}

}  // extern "C"
