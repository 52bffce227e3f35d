// Products with weights held as 4-bit whole numbers, a scale and a zero point for every group of inputs:
//   y[n, o] = sum over k of x[n, k] s[o, k / group] (q[o, k] - z[o, k / group]) + bias[o].
//
// The codes of 16 outputs and 128 inputs (a tile and a span) are 1 KiB: lane (quarter, r) of a wave finds in
// its 16 bytes the inputs 32 j + 8 quarter + (0 .. 7) of output r in word j, as the matrix instructions take
// them.  A code q is the e4m3 number q / 512 (its subnormal numbers and the eight above are evenly
// spaced), so one instruction turns two codes into exact BF16 or FP16 numbers.  Products of codes and x
// are summed in FP32 by group and only then scaled: no weight is rounded.  FP32 inputs are three BF16
// terms that add up to them.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "mf_mx.h"

namespace mf {

typedef f16 v8h __attribute__((ext_vector_type(8)));
typedef f16 v2h __attribute__((ext_vector_type(2)));

constexpr int TILE = 16, SPAN_K = 128, SPAN_BYTES = TILE * SPAN_K / 2;

struct HeldArgs {
    const void *x;          // [n, k], rows ldx apart
    i64 n, k, ldx;
    const u8 *codes;        // [tiles, spans, 1024]
    const void *scales;     // [tiles, groups, 16]
    const u8 *zeros;        // the same, or nullptr: 8
    i64 o, groups, spans;
    int shift;              // log2(group)
    const void *bias;       // [o] or nullptr
    void *out;              // [n, o]
};

// The operand types of the matrix instructions: F16 for FP16 inputs, BF16 for the others.
template <typename T> struct Operand {
    typedef v8bf V;
    static constexpr int TERMS = std::is_same<T, float>::value ? 3 : 1;
    static __device__ __forceinline__ V codes(u32 w) {
        const u32 lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
        v4u r;
        r[0] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, false));
        r[1] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, true));
        r[2] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, false));
        r[3] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, true));
        return __builtin_bit_cast(V, r);
    }
    static __device__ __forceinline__ V ones() {
        v4u r = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
        return __builtin_bit_cast(V, r);
    }
    static __device__ __forceinline__ v4f mfma(V a, V b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};
template <> struct Operand<f16> {
    typedef v8h V;
    static constexpr int TERMS = 1;
    static __device__ __forceinline__ V codes(u32 w) {
        const u32 lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
        v4u r;
        r[0] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.0f, false));
        r[1] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.0f, true));
        r[2] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.0f, false));
        r[3] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.0f, true));
        return __builtin_bit_cast(V, r);
    }
    static __device__ __forceinline__ V ones() {
        v4u r = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
        return __builtin_bit_cast(V, r);
    }
    static __device__ __forceinline__ v4f mfma(V a, V b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};

// x's values in the upper halves of FP32 numbers: what is left of them is exact.
__device__ __forceinline__ float upper(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }

// Eight consecutive values of a row, at a 16-byte address.
template <typename T> struct alignas(16) Eight {
    T v[8];
    __device__ __forceinline__ void load(const T *at) {
#pragma unroll
        for (int i = 0; i < 8; i += PIECE<T>)
            *reinterpret_cast<Piece<T> *>(v + i) = *reinterpret_cast<const Piece<T> *>(at + i);
    }
    // The terms that add up to them.
    template <int TERMS, typename V> __device__ __forceinline__ void split(V (&t)[TERMS]) const {
        if constexpr (TERMS == 1) {
            t[0] = *reinterpret_cast<const V *>(v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float rest = v[i];
#pragma unroll
                for (int n = 0; n < TERMS; ++n) {
                    const float high = upper(rest);
                    t[n][i] = bf16(high);
                    rest -= high;
                }
            }
        }
    }
};

// The wave's number in its workgroup, the same for all its lanes.
__device__ __forceinline__ int wave_of_workgroup() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// The four values that the quarters of a wave hold, each in all of them.
__device__ __forceinline__ void quarters(float value, float (&all)[4]) {
    const u32 v = __float_as_uint(value);
    const auto halves = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    const auto low = __builtin_amdgcn_permlane16_swap(halves[0], halves[0], false, false);
    const auto high = __builtin_amdgcn_permlane16_swap(halves[1], halves[1], false, false);
    all[0] = __uint_as_float(low[0]), all[1] = __uint_as_float(low[1]);
    all[2] = __uint_as_float(high[0]), all[3] = __uint_as_float(high[1]);
}

// ---- few rows --------------------------------------------------------------
// A workgroup takes OT tiles of outputs and all rows, its waves split the spans and add their sums in LDS in
// the order of the waves.  Row 4 i + quarter of a block of 16 rows is row 4 quarter + i of the matrix
// instruction, so that up to 4 rows need one register of its result and one scaling.  x is a multiple of
// 8 inputs wide, in whole 16-byte pieces.  PER: scalings in a span, 1 for groups of 128 on, else 4.
// 1 x 4096 x 11008 BF16, groups of 32, in 7.5 us (25 MB, 3.4 TB/s), 1 x 4096 x 4096, groups of 128, in 3.7, a
// launch: bound by a wave's chain of four or five spans and the 57% of the time that the vector units take for
// conversions and scalings. More rows read x again for every tile from the L2: 16 x 4096 x 11008 12 us. Waves
// a workgroup: 4 / 8 / 16 for the first 7.7 / 7.4 / 8.8 us; x fetched with its span 7.6.
template <typename T, typename S, int WAVES, int OT, int NB, int R, int PER, bool AHEAD>
__global__ __launch_bounds__(64 * WAVES) void k_int4_few(const HeldArgs a) {
    typedef Operand<T> Op;
    constexpr int TERMS = Op::TERMS;
    extern __shared__ __align__(16) float sums[];   // [WAVES][OT * NB * R][64]
    const int lane = threadIdx.x & 63, wave = wave_of_workgroup();
    const int quarter = lane >> 4, r = lane & 15;
    const int spans = int(a.spans), groups = int(a.groups), k = int(a.k);
    const i64 tiles = (a.o + TILE - 1) / TILE, tile0 = i64(blockIdx.x) * OT;
    const T *rows[NB];      // at this lane's eight inputs of the wave's next span
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const i64 n = min(i64(16 * b + (r & 3) * 4 + (r >> 2)), a.n - 1);
        rows[b] = static_cast<const T *>(a.x) + n * a.ldx + wave * SPAN_K + 8 * quarter;
    }

    v4u next[OT];
    S next_s[OT];
    u8 next_z[OT];
    Eight<T> next_x[NB][4];
    const auto fetch_x = [&](int span) {
        if ((span + 1) * SPAN_K <= k) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int j = 0; j < 4; ++j) next_x[b][j].load(rows[b] + 32 * j);
        } else {            // the last span of a row that ends within it: zeros past the end
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bool in = span * SPAN_K + 32 * j + 8 * quarter < k;
                    next_x[b][j].load(in ? rows[b] + 32 * j : rows[b] - span * SPAN_K - 8 * quarter);
#pragma unroll
                    for (int i = 0; i < 8; ++i) next_x[b][j].v[i] = in ? next_x[b][j].v[i] : T(0.0f);
                }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) rows[b] += WAVES * SPAN_K;
    };
    const auto fetch = [&](int span) {
        // A quarter reads the scale of the 32 inputs that are its number.
        const u32 g = PER == 1 ? (span * SPAN_K) >> a.shift
                               : min((span * SPAN_K + 32 * quarter) >> a.shift, groups - 1);
#pragma unroll
        for (int t = 0; t < OT; ++t) {
            const i64 tile = min(tile0 + t, tiles - 1);
            const u8 *at = a.codes + (tile * spans + span) * SPAN_BYTES;
            next[t] = *reinterpret_cast<const v4u *>(at + u32(lane * 16));
            next_s[t] = (static_cast<const S *>(a.scales) + tile * groups * 16)[g * 16 + r];
            next_z[t] = u8(8);
            if (a.zeros) next_z[t] = (a.zeros + tile * groups * 16)[g * 16 + r];
        }
        if (AHEAD) fetch_x(span);
    };

    v4f total[OT][NB];
#pragma unroll
    for (int t = 0; t < OT; ++t)
#pragma unroll
        for (int b = 0; b < NB; ++b) total[t][b] = v4f{0, 0, 0, 0};
    if (wave < spans) fetch(wave);
    for (int span = wave; span < spans; span += WAVES) {
        v4u w[OT];
        Eight<T> x[NB][4];
        float scale[OT][PER], zero[OT][PER];
        if (!AHEAD) fetch_x(span);
#pragma unroll
        for (int t = 0; t < OT; ++t) {
            w[t] = next[t];
            const float s = float(next_s[t]), z = -float(next_z[t]);
            if constexpr (PER == 1) {
                scale[t][0] = s, zero[t][0] = z;
            } else {
                quarters(s, scale[t]);
                quarters(z, zero[t]);
            }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < 4; ++j) x[b][j] = next_x[b][j];
        if (span + WAVES < spans) fetch(span + WAVES);
        v4f acc[OT][NB], sum[NB];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            typename Op::V q[OT];
            constexpr int STEPS = 4 / PER;
#pragma unroll
            for (int t = 0; t < OT; ++t) q[t] = Op::codes(w[t][j]);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                typename Op::V xs[TERMS];
                x[b][j].template split<TERMS>(xs);
                if (j % STEPS == 0) {
                    sum[b] = v4f{0, 0, 0, 0};
#pragma unroll
                    for (int t = 0; t < OT; ++t) acc[t][b] = v4f{0, 0, 0, 0};
                }
#pragma unroll
                for (int m = 0; m < TERMS; ++m) {
                    sum[b] = Op::mfma(xs[m], Op::ones(), sum[b]);
#pragma unroll
                    for (int t = 0; t < OT; ++t) acc[t][b] = Op::mfma(xs[m], q[t], acc[t][b]);
                }
            }
            if ((j + 1) % STEPS == 0)
#pragma unroll
                for (int t = 0; t < OT; ++t)
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int i = 0; i < R; ++i)
                            total[t][b][i] = fmaf(scale[t][j / STEPS],
                                                  fmaf(zero[t][j / STEPS], sum[b][i], acc[t][b][i]),
                                                  total[t][b][i]);
        }
    }
    constexpr int VALUES = OT * NB * R;
#pragma unroll
    for (int t = 0; t < OT; ++t)
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < R; ++i)
                sums[(wave * VALUES + (t * NB + b) * R + i) * 64 + lane] = total[t][b][i];
    __syncthreads();
    for (int v = wave; v < VALUES; v += WAVES) {
        const int t = v / (NB * R), b = v / R % NB, i = v % R;
        const i64 n = 16 * b + 4 * i + quarter, o = (tile0 + t) * TILE + r;
        float y = 0.0f;
#pragma unroll
        for (int u = 0; u < WAVES; ++u) y += sums[(u * VALUES + v) * 64 + lane];
        if (n < a.n && o < a.o) {
            if (a.bias) y += float(static_cast<const T *>(a.bias)[o]);
            static_cast<T *>(a.out)[n * a.o + o] = rounded<T>(y);
        }
    }
}

// Copies rows of x into rows of whole spans, with zeros past k: one wave a span, two inputs a lane. For few rows
// that are not whole 16-byte pieces; bound by its launch.
template <typename T>
__global__ __launch_bounds__(256) void k_int4_pad(const T *x, i64 n, i64 k, i64 ldx, i64 spans, T *out) {
    const int lane = threadIdx.x & 63;
    for (i64 id = i64(blockIdx.x) * 4 + (threadIdx.x >> 6); id < n * spans; id += i64(gridDim.x) * 4) {
        const i64 row = id / spans, span = id - row * spans;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const i64 at = span * SPAN_K + lane * 2 + i;
            out[row * spans * SPAN_K + at] = at < k ? x[row * ldx + at] : T(0.0f);
        }
    }
}

// ---- many rows -------------------------------------------------------------
// Rows of x as the tile kernel copies them, and their sums: [blocks, pitch] of `factor` times the sum of each
// row over a block of 32 inputs (`per` 4 to a span), 64 (2) or 128 (1), 0 past the rows.
struct PrepareArgs {
    const void *x;
    i64 n, k, ldx, spans, pitch;
    int per;
    float factor;
    float *sums;        // or nullptr
    u16 *planes;        // [TERMS, n, 128 spans], or nullptr: x is taken as it is
};

// A workgroup takes 16 spans of a row, a lane eight inputs. Bound by its bytes and launch: 2048 x 4096 BF16 in
// 5 us (17 MB).
template <typename T, bool PIECES> __global__ __launch_bounds__(256) void k_int4_prepare(const PrepareArgs a) {
    typedef typename std::conditional<std::is_same<T, float>::value, bf16, T>::type Term;
    constexpr int TERMS = Operand<T>::TERMS;
    const i64 n = blockIdx.y, span = i64(blockIdx.x) * 16 + (threadIdx.x >> 4);
    const int piece = threadIdx.x & 15;
    if (span >= a.spans) return;
    Eight<T> x;
#pragma unroll
    for (int i = 0; i < 8; ++i) x.v[i] = T(0.0f);
    if (n < a.n) {
        const i64 k = span * SPAN_K + piece * 8;
        const T *row = static_cast<const T *>(a.x) + n * a.ldx;
        if (PIECES && k + 8 <= a.k) {
            x.load(row + k);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (k + i < a.k) x.v[i] = row[k + i];
        }
        if (a.planes) {
            alignas(16) Term terms[TERMS][8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float rest = float(x.v[i]);
#pragma unroll
                for (int t = 0; t < TERMS; ++t) {
                    const float high = TERMS == 1 ? rest : upper(rest);
                    terms[t][i] = Term(high);
                    rest -= high;
                }
            }
#pragma unroll
            for (int t = 0; t < TERMS; ++t)
                *reinterpret_cast<v4u *>(a.planes + ((t * a.n + n) * a.spans * SPAN_K + k)) =
                    *reinterpret_cast<const v4u *>(terms[t]);
        }
    }
    if (!a.sums) return;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += float(x.v[i]);
    sum += __shfl_xor(sum, 1);
    sum += __shfl_xor(sum, 2);
    if (a.per < 4) sum += __shfl_xor(sum, 4);
    if (a.per < 2) sum += __shfl_xor(sum, 8);
    const int shift = a.per == 4 ? 2 : a.per == 2 ? 3 : 4;     // log2 of a block's pieces
    if ((piece & ((1 << shift) - 1)) == 0) a.sums[(span * a.per + (piece >> shift)) * a.pitch + n] = a.factor * sum;
}

struct TileArgs {
    HeldArgs h;             // h.x: rows of 16-bit operands, h.ldx apart, of whole spans
    i64 plane;              // distance of x's terms, in values
    const float *sums;      // x's sums, or (TABLE false) nullptr
    i64 pitch;
    i64 splits, share;      // workgroups along the spans, and the spans of each
    float *parts;           // [splits, n, o], where there are several
};

template <typename T> __device__ __forceinline__ v16f mfma_wide(v4u a, v4u b, v16f c) {
    if constexpr (std::is_same<T, f16>::value)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b),
                                                      c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a),
                                                       __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}

// A workgroup of four waves takes 32 NT rows and 128 NO outputs, a wave 32 NO of them: its codes go from
// memory to registers, where they become operands once for all rows; x comes through LDS, copied by DMA a
// span ahead.  With the sums' TABLE, sums over a group begin at -8 times the sum of x, so a zero point of 8
// costs nothing; others (ZEROS) are taken off with one operation more a group and result, the sums read when
// they are (held from the group's start, with zero points and groups of 32, BF16 takes 359 us for 318 and FP16
// 442 for 344).  Without it a matrix instruction with ones gives the sums.  PER: scalings in a span, 1 for
// groups of 128 on, 2 for 64, 4 for 32 (2048 x 4096 x 11008 BF16 with groups of 64: four 250 us, two 210; 24 x
// 11008 x 4096 18 and 16).  A third of the variants spill up to 16 registers, nearly all outside the span's loop
// (FP32 in tiles of 64 by 128 with groups of 32 reads nine back a span, three others one).
// 2048 x 4096 x 11008 BF16, groups of 128, in 181 us (1020 TFLOP/s). No one unit bounds it: matrix units are busy
// 54% of the time and vector issue 59%, and of two waves a SIMD each waits for a busy unit 40% of its time and for a
// stage 17%. Without conversions, scalings and LDS reads the loop takes 182 too, not the matrix units' 110; tiles
// of 128 rows, one wave a SIMD, take 265, with the whole span's codes converted first it is the same. Groups of
// 32, four scalings a span, 245: the vector units. In small tiles a span's copies are waited for (24 x 11008 x
// 4096 FP16 11 us); four stages of them with the codes among them leave one workgroup a compute unit and take 15.
constexpr int TILE_WAVES = 4, BAND = 8;

// Waves that a SIMD has to hold: with at most 256 registers each the matrix instructions' results stay where
// the vector units reach them (else each is copied once more for its scaling).
constexpr int tile_waves_per_simd(int nt, int no) { return nt * no == 1 ? 4 : nt * no == 2 ? 3 : 2; }

template <typename T, typename S, int NT, int NO, bool TABLE, bool ZEROS, int PER>
__global__ __launch_bounds__(64 * TILE_WAVES, tile_waves_per_simd(NT, NO)) void
k_int4_tile(const TileArgs t) {
    static_assert(TABLE || ZEROS, "sums that begin at 0 have the zero points taken off");
    typedef Operand<T> Op;
    constexpr int TERMS = Op::TERMS, ROWS = 32 * NT, OUTPUTS = 32 * NO * TILE_WAVES;
    constexpr int XBYTES = TERMS * ROWS * SPAN_K * 2, STAGE = XBYTES + (TABLE ? 2048 : 0);
    extern __shared__ __align__(16) u8 staged[];
    const HeldArgs &a = t.h;
    const int lane = threadIdx.x & 63, wave = wave_of_workgroup();
    const int half = lane >> 5, row = lane & 31, r = lane & 15;
    const u32 tn = u32((a.n + ROWS - 1) / ROWS), to = u32((a.o + OUTPUTS - 1) / OUTPUTS);
    // Each XCD takes a run of tiles (xcd_tile), here in bands of BAND tiles of rows and all outputs, so that what
    // it reads at a time is as much of x as of W and stays in its L2.
    u32 nx, oy;
    xcd_tile(blockIdx.x, 1, tn * to * u32(t.splits), nx, oy);
    const u32 columns = to * u32(t.splits), band = oy / (BAND * columns), within = oy - band * BAND * columns;
    const u32 high = min(u32(BAND), tn - band * BAND);
    nx = band * BAND + within % high;
    oy = within / high;
    const u32 split = oy % u32(t.splits);
    const i64 n0 = i64(nx) * ROWS, o0 = i64(oy / u32(t.splits)) * OUTPUTS + wave * (32 * NO);
    const i64 tiles = (a.o + TILE - 1) / TILE;
    const int first = int(split * t.share), last = int(min(first + t.share, a.spans));

    // Copies: 1 KiB each, four rows of x (row q's 16-byte pieces p at p ^ (q & 15)) or two rows of sums.
    constexpr int COPIES = XBYTES / 1024 / TILE_WAVES;
    const char *source[COPIES];
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
        const int q = (wave * COPIES + i) * 4 + (lane >> 4);        // a row of a term
        const i64 n = min(n0 + q % ROWS, a.n - 1);
        source[i] = static_cast<const char *>(a.x) +
                    (i64(q / ROWS) * t.plane + n * a.ldx + (((lane & 15) ^ (q & 15)) * 8)) * 2;
    }
    const float *sums = t.sums + n0 + (lane & 31) * 4;
    const u32 lds = lds_address(staged);
    const auto copy = [&](int span) {
        const u32 to = lds + (span & 1) * STAGE;
#pragma unroll
        for (int i = 0; i < COPIES; ++i)
            lds_dma_16(source[i] + i64(span) * (SPAN_K * 2),
                       __builtin_amdgcn_readfirstlane(to + (wave * COPIES + i) * 1024));
        if (TABLE && wave < (PER + 1) / 2)
            lds_dma_16(sums + i64(span * PER + min(wave * 2 + half, PER - 1)) * t.pitch,
                       __builtin_amdgcn_readfirstlane(to + XBYTES + wave * 1024));
    };

    // A lane's output is 32 j + row of the wave's; it reads both 16-byte pieces of its half.
    const u8 *codes[NO];
    const S *scales[NO];
    const u8 *zeros[NO];
#pragma unroll
    for (int j = 0; j < NO; ++j) {
        const i64 tile = min((o0 + 32 * j + row) / TILE, tiles - 1);
        codes[j] = a.codes + tile * a.spans * SPAN_BYTES + half * 256 + r * 16;
        scales[j] = static_cast<const S *>(a.scales) + tile * a.groups * 16 + r;
        zeros[j] = ZEROS && a.zeros ? a.zeros + tile * a.groups * 16 + r : nullptr;
    }
    v4u w[NO][2];
    S s[NO][PER];
    u8 z[NO][PER];
    const auto fetch = [&](int span) {
#pragma unroll
        for (int j = 0; j < NO; ++j) {
#pragma unroll
            for (int m = 0; m < 2; ++m)
                w[j][m] = *reinterpret_cast<const v4u *>(codes[j] + i64(span) * SPAN_BYTES + m * 512);
#pragma unroll
            for (int g = 0; g < PER; ++g) {
                const int at = min((span * SPAN_K + g * (SPAN_K / PER)) >> a.shift, int(a.groups) - 1) * 16;
                s[j][g] = scales[j][at];
                z[j][g] = u8(8);
                if (ZEROS && a.zeros) z[j][g] = zeros[j][at];
            }
        }
    };

    // The staged sums of group g of a span for this lane's results of 32 rows.
    const auto read_sums = [&](const u8 *stage, int g, int i, v16f &to) {
        const float *from = reinterpret_cast<const float *>(stage + XBYTES) + g * 128 + 32 * i + 4 * half;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const v4f four = *reinterpret_cast<const v4f *>(from + 8 * e);
#pragma unroll
            for (int f = 0; f < 4; ++f) to[4 * e + f] = four[f];
        }
    };

    v16f total[NT][NO] = {};
    if (first < last) {
        fetch(first);
        copy(first);
    }
    for (int span = first; span < last; ++span) {
        wait_stage<0>();
        if (span + 1 < last) copy(span + 1);
        const u8 *stage = staged + (span & 1) * STAGE;
        v4u held[NO][2];
        float scale[NO][PER], zero[NO][PER];
#pragma unroll
        for (int j = 0; j < NO; ++j) {
#pragma unroll
            for (int m = 0; m < 2; ++m) held[j][m] = w[j][m];
#pragma unroll
            for (int g = 0; g < PER; ++g) scale[j][g] = float(s[j][g]), zero[j][g] = -float(z[j][g]);
        }
        if (span + 1 < last) fetch(span + 1);
        v16f acc[NT][NO], sum[NT];
#pragma unroll
        for (int b = 0; b < 8; ++b) {       // 16 inputs each
            constexpr int STEPS = 8 / PER;
            v4u q[NO];
#pragma unroll
            for (int j = 0; j < NO; ++j) q[j] = __builtin_bit_cast(v4u, Op::codes(held[j][b & 1][b >> 1]));
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                if (b % STEPS == 0) {
                    if (TABLE && !ZEROS) read_sums(stage, b / STEPS, i, sum[i]);
                    else sum[i] = v16f{};
#pragma unroll
                    for (int j = 0; j < NO; ++j) acc[i][j] = ZEROS ? v16f{} : sum[i];
                }
#pragma unroll
                for (int m = 0; m < TERMS; ++m) {
                    const v4u xf = *reinterpret_cast<const v4u *>(
                        stage + (m * ROWS + 32 * i + row) * (SPAN_K * 2) + ((2 * b + half) ^ r) * 16);
#pragma unroll
                    for (int j = 0; j < NO; ++j) acc[i][j] = mfma_wide<T>(xf, q[j], acc[i][j]);
                    if (!TABLE) sum[i] = mfma_wide<T>(xf, __builtin_bit_cast(v4u, Op::ones()), sum[i]);
                }
            }
            if ((b + 1) % STEPS == 0)
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    if (TABLE && ZEROS) read_sums(stage, b / STEPS, i, sum[i]);
#pragma unroll
                    for (int j = 0; j < NO; ++j)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float v =
                                ZEROS ? fmaf(zero[j][b / STEPS], sum[i][e], acc[i][j][e]) : acc[i][j][e];
                            total[i][j][e] = fmaf(scale[j][b / STEPS], v, total[i][j][e]);
                        }
                }
        }
    }
#pragma unroll
    for (int j = 0; j < NO; ++j) {
        const i64 o = o0 + 32 * j + row;
        if (o >= a.o) continue;
        const float bias = a.bias && t.splits == 1 ? float(static_cast<const T *>(a.bias)[o]) : 0.0f;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const i64 n = n0 + 32 * i + 8 * (e / 4) + 4 * half + (e & 3);
                if (n >= a.n) continue;
                if (t.splits > 1)
                    t.parts[(split * a.n + n) * a.o + o] = total[i][j][e];
                else
                    static_cast<T *>(a.out)[n * a.o + o] = rounded<T>(total[i][j][e] + bias);
            }
    }
}

// Adds the parts of a product in their order, and the bias. Bound by its launch (2 to 4 us).
template <typename T> __global__ __launch_bounds__(256) void k_int4_join(const TileArgs t) {
    const i64 all = t.h.n * t.h.o;
    for (i64 id = i64(blockIdx.x) * 256 + threadIdx.x; id < all; id += i64(gridDim.x) * 256) {
        float y = 0.0f;
        for (i64 s = 0; s < t.splits; s += 8) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = t.parts[min(s + i, t.splits - 1) * all + id];
#pragma unroll
            for (int i = 0; i < 8; ++i) y += s + i < t.splits ? v[i] : 0.0f;
        }
        if (t.h.bias) y += float(static_cast<const T *>(t.h.bias)[id % t.h.o]);
        static_cast<T *>(t.h.out)[id] = rounded<T>(y);
    }
}

// ---------------------------------------------------------------------------
// Quantization
// ---------------------------------------------------------------------------
struct Int4QuantizeArgs {
    const void *w;      // [o, k], rows ldw apart
    i64 o, k, ldw, groups, spans;
    int shift;
    u8 *codes;
    void *scales;
};

// A wave works on 512 inputs of an output, eight a lane: the four bytes of codes that a lane's word of a tile is.
constexpr int WAVE_INPUTS = 512;

// Where the codes of output o and inputs k to k + 7 lie.
__device__ __forceinline__ i64 word_of(i64 o, i64 k, i64 spans) {
    const int in = int(k) & (SPAN_K - 1);
    return ((o / TILE) * spans + (k >> 7)) * SPAN_BYTES + (in >> 3 & 3) * 256 + (o & 15) * 16 + (in >> 5) * 4;
}

// The peak of each group, the scale peak / 7 in the scales' type, and the codes round(w / scale) + 8. A group of more
// than 512 inputs is read twice. It runs once a weight: 11008 x 4096 BF16 in 52 us (113 MB, 2.2 TB/s).
// Its words are 16 bytes apart in a tile, which the L2 joins.
template <typename T, typename S, bool PIECES>
__global__ __launch_bounds__(256) void k_int4_quantize(const Int4QuantizeArgs a) {
    const int lane = threadIdx.x & 63;
    const i64 step = std::max<i64>(WAVE_INPUTS, i64(1) << a.shift), padded = a.spans * SPAN_K;
    const i64 chunks = (padded + step - 1) / step, all = (a.o + TILE - 1) / TILE * TILE * chunks;
    const int lanes = a.shift >= 9 ? 64 : 1 << (a.shift - 3);       // of a group
    for (i64 id = i64(blockIdx.x) * 4 + wave_of_workgroup(); id < all; id += i64(gridDim.x) * 4) {
        const i64 o = id / chunks, first = (id - o * chunks) * step + lane * 8;
        const i64 end = min(first - lane * 8 + step, padded);
        const T *w = static_cast<const T *>(a.w) + o * a.ldw;
        Eight<T> v;
        const auto load = [&](i64 k) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v.v[i] = T(0.0f);
            if (o >= a.o) return;
            if (PIECES && k + 8 <= a.k) {
                v.load(w + k);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (k + i < a.k) v.v[i] = w[k + i];
            }
        };
        float peak = 0.0f;
        bool bad = false;
        for (i64 k = first; k < end; k += WAVE_INPUTS) {
            load(k);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float size = fabsf(float(v.v[i]));
                bad |= !(size <= FLT_MAX);
                peak = fmaxf(peak, size);
            }
        }
        for (int d = lanes >> 1; d; d >>= 1) {
            peak = fmaxf(peak, __shfl_xor(peak, d));
            bad |= __shfl_xor(int(bad), d) != 0;
        }
        S held = S(peak > 0.0f ? peak / 7.0f : 1.0f);
        if (peak > 0.0f && !(float(held) > 0.0f)) held = S(1.0f);     // beneath the type: codes of 0
        if (bad) held = S(NAN);
        const i64 g = first >> a.shift;
        if ((lane & (lanes - 1)) == 0 && g < a.groups)
            static_cast<S *>(a.scales)[(o / TILE * a.groups + g) * 16 + (o & 15)] = o < a.o ? held : S(0.0f);
        for (i64 k = first; k < end; k += WAVE_INPUTS) {
            if (step > WAVE_INPUTS) load(k);
            u32 word = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float c = bad ? 0.0f : rintf(float(v.v[i]) / float(held));
                c = fminf(fmaxf(c, -8.0f), 7.0f);
                word |= u32(int(c) + 8) << (8 * (i & 3) + (i & 4));
            }
            *reinterpret_cast<u32 *>(a.codes + word_of(o, k, a.spans)) = word;
        }
    }
}

// A lane restores eight values: 11008 x 4096 to BF16 in 50 us.
template <typename T, typename S, bool PIECES>
__global__ __launch_bounds__(256) void k_int4_dequantize(const HeldArgs a) {
    const int lane = threadIdx.x & 63;
    const i64 chunks = (a.k + WAVE_INPUTS - 1) / WAVE_INPUTS, all = a.o * chunks;
    for (i64 id = i64(blockIdx.x) * 4 + wave_of_workgroup(); id < all; id += i64(gridDim.x) * 4) {
        const i64 o = id / chunks, k = (id - o * chunks) * WAVE_INPUTS + lane * 8;
        if (k >= a.k) continue;
        const u32 word = *reinterpret_cast<const u32 *>(a.codes + word_of(o, k, a.spans));
        const i64 g = (o / TILE * a.groups + (k >> a.shift)) * 16 + (o & 15);   // eight inputs are of one group
        const float scale = float(static_cast<const S *>(a.scales)[g]), zero = a.zeros ? float(a.zeros[g]) : 8.0f;
        alignas(16) T v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = rounded<T>(scale * (float(word >> (8 * (i & 3) + (i & 4)) & 15u) - zero));
        T *out = static_cast<T *>(a.out) + o * a.k + k;
        if (PIECES && k + 8 <= a.k) {
#pragma unroll
            for (int i = 0; i < 8; i += PIECE<T>)
                *reinterpret_cast<Piece<T> *>(out + i) = *reinterpret_cast<const Piece<T> *>(v + i);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (k + i < a.k) out[i] = v[i];
        }
    }
}

// log2 of a group that is a power of two of at least 32, or -1.
int group_shift(i64 group) {
    for (int s = 5; s <= 24; ++s)
        if (group == i64(1) << s) return s;
    return -1;
}

constexpr i64 MOST_OUTPUTS = i64(1) << 25, MOST_INPUTS = i64(1) << 24, MOST_ROWS = i64(1) << 27;

int check_held(const void *codes, const void *scales, int32_t scale_type, const void *zeros, i64 o, i64 k,
               i64 group, HeldArgs &a) {
    if (!codes || !scales || !known_type(scale_type) || o < 1 || k < 1 || group_shift(group) < 0)
        return fail(MF_E_INVALID, "invalid 4-bit weight");
    if (o >= MOST_OUTPUTS || k >= MOST_INPUTS)
        return fail(MF_E_UNSUPPORTED, "4-bit weight of %lld outputs and %lld inputs", (long long)o,
                    (long long)k);
    if (!aligned(codes, 16) || !aligned(scales, type_bytes(scale_type)))
        return fail(MF_E_INVALID, "4-bit weight is not aligned");
    a.codes = static_cast<const u8 *>(codes);
    a.scales = scales;
    a.zeros = static_cast<const u8 *>(zeros);
    a.o = o, a.k = k, a.shift = group_shift(group);
    a.groups = (k + group - 1) >> a.shift;
    a.spans = (k + SPAN_K - 1) / SPAN_K;
    return MF_OK;
}

template <typename T, typename S, int OT, int NB, int R> int launch_few(const HeldArgs &a, hipStream_t s) {
    // x a span ahead, where there are registers for it.
    constexpr int WAVES = 8;
    constexpr bool AHEAD = Operand<T>::TERMS == 1 || NB < 3;
    const i64 tiles = (a.o + TILE - 1) / TILE;
    const int lds = WAVES * OT * NB * R * 64 * int(sizeof(float));
    const auto kernel = a.shift >= 7 ? k_int4_few<T, S, WAVES, OT, NB, R, 1, AHEAD>
                                     : k_int4_few<T, S, WAVES, OT, NB, R, 4, AHEAD>;
    const int status = allow_lds(kernel, lds);
    if (status) return status;
    hipLaunchKernelGGL(kernel, dim3(u32((tiles + OT - 1) / OT)), dim3(64 * WAVES), lds, s, a);
    return check_launch("4-bit product");
}

constexpr i64 ROWS_AT_ONCE = 8192;

// The kernel, how many rows go through tiles at a time, and what the workspace holds for them.
struct HeldPlan {
    enum { FEW, MID, LARGE } kernel;
    bool direct;            // x is read as it is
    int32_t type;
    int per, terms;
    i64 rows, pitch, spans, sums, planes, splits = 1, share, bytes;
    HeldPlan(int32_t type, i64 n, i64 k, i64 o, i64 group, bool pieces) : type(type) {
        spans = share = (k + SPAN_K - 1) / SPAN_K;
        per = group >= SPAN_K ? 1 : int(SPAN_K / group);
        terms = type == MF_F32 ? 3 : 1;
        rows = std::min(n, ROWS_AT_ONCE);
        kernel = few(type, n, k, o) ? FEW : large(type, rows, o) ? LARGE : MID;
        direct = kernel == FEW ? pieces && k % 8 == 0 : pieces && type != MF_F32 && k % SPAN_K == 0;
        pitch = (rows + 127) / 128 * 128 + 128;
        sums = kernel == LARGE ? spans * per * pitch * i64(sizeof(float)) : 0;
        planes = direct ? 0 : rows * spans * SPAN_K * (kernel == FEW ? type_bytes(type) : 2 * terms);
        if (kernel != FEW) {
            // Spans are split until every compute unit has a workgroup, or two of those of 32 rows that
            // scale four times a span (us, 64 x 4096 x 4096, groups of 128, 8 / 12 / 16 splits: 15 / 19 / 20;
            // 24 x 11008 x 4096, 8 / 16: 14 / 15; 32 x 4096 x 11008, groups of 32, 2 / 5: 26 / 20).
            const i64 tiles = kernel == LARGE ? large_tiles(rows, o)
                                              : (rows + mid_rows(n) - 1) / mid_rows(n) * ((o + 127) / 128);
            const i64 wanted = kernel == LARGE ? 256 / tiles : ((per == 1 ? 256 : 512) + tiles - 1) / tiles;
            if (std::min(wanted, spans / 2) > 1) {
                share = (spans + std::min(wanted, spans / 2) - 1) / std::min(wanted, spans / 2);
                splits = (spans + share - 1) / share;
            }
        }
        bytes = sums + planes + (splits > 1 ? splits * rows * o * i64(sizeof(float)) : 0);
    }
    // Workgroups of k_int4_few read all of x again for every tile, or for two (wide).
    static bool wide(i64 n, i64 o) { return n > 4 && n <= 32 && o >= 8192; }
    // Up to 64 rows while that is little, and a wave's chain of spans short (us, few / tiles: 24 x 4096 x
    // 4096 8.9 / 13.3, 48 x 2048 x 2048 8.0 / 8.9, 24 x 11008 x 4096 20 / 14, 64 x 4096 x 1024 17 / 11,
    // 32 x 4096 x 11008 20 / 16).
    static bool few(int32_t type, i64 n, i64 k, i64 o) {
        const i64 tiles = (o + TILE - 1) / TILE / (wide(n, o) ? 2 : 1);
        return n <= 16 || (n <= 64 && (k + SPAN_K - 1) / SPAN_K * ((n + 15) / 16) <= 64 &&
                           tiles * n * k * type_bytes(type) <= i64(72) << 20);
    }
    static i64 mid_rows(i64 n) { return n <= 32 ? 32 : 64; }
    static i64 large_tiles(i64 n, i64 o) { return (n + 63) / 64 * ((o + 255) / 256); }
    // The sums' launch and the wide tiles pay for many rows where they are tiles enough (us, mid / large: 256 x
    // 4096 x 11008 47 / 41, 128 of them 31 / 30, 256 x 4096 x 4096 31 / 30, 300 x 2048 x 2048 16 / 19, 512 x 4096
    // x 1024 21 / 26). FP32 has a launch before its tiles anyway and sums that take three times the instructions:
    // from fewer on (70 x 11008 x 4096 87 / 48, 40 x 4096 x 11008 72 / 33, 100 x 4096 x 2048 33 / 26, 64 x
    // 4096 x 4096 34 / 27; 100 x 1024 x 2048 17 / 18; 77 x 1500 x 1111, ten tiles, 17 / 18).
    static bool large(int32_t type, i64 n, i64 o) {
        return type == MF_F32 ? n > 32 && o > 128 && large_tiles(n, o) >= 16
                              : n > 128 && o > 128 && large_tiles(n, o) >= 64;
    }
};

bool rows_in_pieces(const void *x, i64 ldx, int32_t type) {
    return aligned(x, 16) && ldx * type_bytes(type) % 16 == 0;
}

template <typename T, typename S, int NT, int NO, bool TABLE, bool ZEROS, int PER>
int launch_tile(const TileArgs &t, hipStream_t s) {
    constexpr int ROWS = 32 * NT, OUTPUTS = 32 * NO * TILE_WAVES;
    constexpr int LDS = 2 * (Operand<T>::TERMS * ROWS * SPAN_K * 2 + (TABLE ? 2048 : 0));
    const auto kernel = k_int4_tile<T, S, NT, NO, TABLE, ZEROS, PER>;
    const int status = allow_lds(kernel, LDS);
    if (status) return status;
    const i64 tiles = (t.h.n + ROWS - 1) / ROWS * ((t.h.o + OUTPUTS - 1) / OUTPUTS) * t.splits;
    hipLaunchKernelGGL(kernel, dim3(u32(tiles)), dim3(64 * TILE_WAVES), LDS, s, t);
    return check_launch("4-bit product");
}

// Calls f(PER) for 1, 2 or 4 scalings in a span.
template <typename F> int with_per(int per, F f) {
    return per == 1   ? f(std::integral_constant<int, 1>{})
           : per == 2 ? f(std::integral_constant<int, 2>{})
                      : f(std::integral_constant<int, 4>{});
}

// Tiles of 64 rows and 256 outputs.
template <typename T, typename S> int launch_large(const TileArgs &t, int per, hipStream_t s) {
    return with_per(per, [&](auto p) {
        constexpr int PER = decltype(p)::value;
        return t.h.zeros ? launch_tile<T, S, 2, 2, true, true, PER>(t, s)
                         : launch_tile<T, S, 2, 2, true, false, PER>(t, s);
    });
}

// Tiles of 32 or 64 rows and 128 outputs, with the spans split.
template <typename T, typename S> int launch_mid(const TileArgs &t, int per, hipStream_t s) {
    return with_per(per, [&](auto p) {
        constexpr int PER = decltype(p)::value;
        return HeldPlan::mid_rows(t.h.n) == 32 ? launch_tile<T, S, 1, 1, false, true, PER>(t, s)
                                               : launch_tile<T, S, 2, 1, false, true, PER>(t, s);
    });
}

template <typename T> int launch_join(const TileArgs &t, hipStream_t s) {
    hipLaunchKernelGGL(k_int4_join<T>, dim3(u32(std::min<i64>((t.h.n * t.h.o + 255) / 256, 1 << 16))),
                       dim3(256), 0, s, t);
    return check_launch("4-bit product's parts");
}

template <typename T, typename S>
int launch_tiles(HeldArgs a, const HeldPlan &plan, void *workspace, hipStream_t s) {
    const char *x = static_cast<const char *>(a.x);
    char *out = static_cast<char *>(a.out), *work = static_cast<char *>(workspace);
    const i64 n = a.n;
    for (i64 first = 0; first < n; first += plan.rows) {
        a.n = std::min(plan.rows, n - first);
        a.out = out + first * a.o * i64(sizeof(T));
        a.x = x + first * a.ldx * i64(sizeof(T));
        const bool table = plan.kernel == HeldPlan::LARGE;
        PrepareArgs p{a.x, a.n, a.k, a.ldx, a.spans, table ? plan.pitch : a.n, plan.per,
                      a.zeros ? 1.0f : -8.0f, table ? reinterpret_cast<float *>(work) : nullptr, nullptr};
        TileArgs t{a, 0, p.sums, plan.pitch, plan.splits, plan.share,
                   reinterpret_cast<float *>(work + plan.sums + plan.planes)};
        if (!plan.direct) {
            p.planes = reinterpret_cast<u16 *>(work + plan.sums);
            t.h.x = p.planes;
            t.h.ldx = a.spans * SPAN_K;
            t.plane = a.n * t.h.ldx;
        }
        int status = MF_OK;
        if (table || !plan.direct) {
            const auto prepare = rows_in_pieces(a.x, a.ldx, plan.type) ? k_int4_prepare<T, true>
                                                                        : k_int4_prepare<T, false>;
            hipLaunchKernelGGL(prepare, dim3(u32((a.spans + 15) / 16), u32(p.pitch)), dim3(256), 0, s, p);
            status = check_launch("4-bit product's rows");
        }
        if (!status) status = table ? launch_large<T, S>(t, plan.per, s) : launch_mid<T, S>(t, plan.per, s);
        if (!status && plan.splits > 1) status = launch_join<T>(t, s);
        if (status) return status;
    }
    return MF_OK;
}

template <typename T, typename S> int launch_held(HeldArgs a, const HeldPlan &plan, void *workspace,
                                                  hipStream_t s) {
    if (plan.kernel != HeldPlan::FEW) return launch_tiles<T, S>(a, plan, workspace, s);
    if (!plan.direct) {
        T *rows = static_cast<T *>(workspace);
        hipLaunchKernelGGL(k_int4_pad<T>, dim3(u32((a.n * a.spans + 3) / 4)), dim3(256), 0, s,
                           static_cast<const T *>(a.x), a.n, a.k, a.ldx, a.spans, rows);
        const int status = check_launch("4-bit product's rows");
        if (status) return status;
        a.x = rows;
        a.ldx = a.spans * SPAN_K;
        a.k = a.ldx;        // zeros included: the codes past the weight's inputs are there too
    }
    // Two tiles a workgroup halve what is read of x, and the workgroups: 8 x 4096 x 11008 10.9 -> 9.8 us,
    // 16 of them 14.2 -> 11.7; 16 x 4096 x 4096 6.5 -> 6.7, 1 x 4096 x 4096 3.7 -> 5.1.
    const bool wide = HeldPlan::wide(a.n, a.o);
    return a.n <= 4    ? launch_few<T, S, 1, 1, 1>(a, s)
           : a.n <= 8  ? wide ? launch_few<T, S, 2, 1, 2>(a, s) : launch_few<T, S, 1, 1, 2>(a, s)
           : a.n <= 16 ? wide ? launch_few<T, S, 2, 1, 4>(a, s) : launch_few<T, S, 1, 1, 4>(a, s)
           : a.n <= 32 ? wide ? launch_few<T, S, 2, 2, 4>(a, s) : launch_few<T, S, 1, 2, 4>(a, s)
           : a.n <= 48 ? launch_few<T, S, 1, 3, 4>(a, s)
                       : launch_few<T, S, 1, 4, 4>(a, s);
}

// Calls f(T{}, S{}) for the types of x and of the scales: x's own or FP32.
template <typename F> int with_types(int32_t type, int32_t scale_type, F f) {
    return with_type(type, [&](auto x) {
        using T = decltype(x);
        if (scale_type == MF_F32) return f(x, float{});
        if constexpr (!std::is_same<T, float>::value)
            if (scale_type == type) return f(x, T{});
        return fail(MF_E_INVALID, "scales have to be FP32 or of the operand's type");
    });
}

}  // namespace mf

using namespace mf;

extern "C" {

int mf_int4_quantize(const void *w, int32_t type, int64_t o, int64_t k, int64_t ldw, int64_t group,
                     uint8_t *codes, void *scales, int32_t scale_type, void *stream) {
    HeldArgs h{};
    const int status = check_held(codes, scales, scale_type, nullptr, o, k, group, h);
    if (status) return status;
    if (!w || !known_type(type) || ldw < 0 || (o > 1 && ldw < k) || !aligned(w, type_bytes(type)))
        return fail(MF_E_INVALID, "invalid 4-bit quantization arguments");
    const Int4QuantizeArgs a{w, o, k, ldw, h.groups, h.spans, h.shift, codes, scales};
    const i64 step = std::max<i64>(WAVE_INPUTS, group);
    const i64 waves = (o + TILE - 1) / TILE * TILE * ((h.spans * SPAN_K + step - 1) / step);
    const u32 grid = u32(std::min<i64>((waves + 3) / 4, i64(1) << 20));
    const bool pieces = rows_in_pieces(w, o > 1 ? ldw : 0, type);
    return with_types(type, scale_type, [&](auto x, auto scale) {
        typedef decltype(x) T;
        typedef decltype(scale) S;
        hipLaunchKernelGGL((pieces ? k_int4_quantize<T, S, true> : k_int4_quantize<T, S, false>), dim3(grid),
                           dim3(256), 0, static_cast<hipStream_t>(stream), a);
        return check_launch("4-bit quantization");
    });
}

int mf_int4_dequantize(const uint8_t *codes, const void *scales, int32_t scale_type, const uint8_t *zeros,
                       int64_t o, int64_t k, int64_t group, void *out, int32_t type, void *stream) {
    HeldArgs a{};
    const int status = check_held(codes, scales, scale_type, zeros, o, k, group, a);
    if (status) return status;
    if (!out || !known_type(type) || !aligned(out, type_bytes(type)))
        return fail(MF_E_INVALID, "invalid 4-bit dequantization arguments");
    a.out = out;
    const i64 waves = o * ((k + WAVE_INPUTS - 1) / WAVE_INPUTS);
    const u32 grid = u32(std::min<i64>((waves + 3) / 4, i64(1) << 20));
    const bool pieces = rows_in_pieces(out, o > 1 ? k : 0, type);
    return with_type(type, [&](auto x) {
        return with_type(scale_type, [&](auto scale) {
            typedef decltype(x) T;
            typedef decltype(scale) S;
            hipLaunchKernelGGL((pieces ? k_int4_dequantize<T, S, true> : k_int4_dequantize<T, S, false>),
                               dim3(grid), dim3(256), 0, static_cast<hipStream_t>(stream), a);
            return check_launch("4-bit dequantization");
        });
    });
}

int mf_int4_linear_workspace(int32_t type, int64_t n, int64_t k, int64_t o, int64_t group, int32_t pieces,
                             int64_t *bytes) {
    if (!known_type(type) || n < 1 || k < 1 || o < 1 || n >= MOST_ROWS || k >= MOST_INPUTS ||
        o >= MOST_OUTPUTS || group_shift(group) < 0 || !bytes)
        return fail(MF_E_INVALID, "invalid 4-bit product sizes");
    *bytes = HeldPlan(type, n, k, o, group, pieces != 0).bytes;
    return MF_OK;
}

int mf_int4_linear(const void *x, int32_t type, int64_t n, int64_t k, int64_t ldx, const uint8_t *codes,
                   const void *scales, int32_t scale_type, const uint8_t *zeros, int64_t o, int64_t group,
                   const void *bias, void *out, void *workspace, int64_t bytes, void *stream) {
    HeldArgs a{};
    const int status = check_held(codes, scales, scale_type, zeros, o, k, group, a);
    if (status) return status;
    if (!x || !known_type(type) || n < 1 || ldx < 0 || (n > 1 && ldx < k) || !out)
        return fail(MF_E_INVALID, "invalid 4-bit product arguments");
    const uintptr_t one = type_bytes(type);
    if (!aligned(x, one) || !aligned(bias, one) || !aligned(out, one))
        return fail(MF_E_INVALID, "4-bit product's operands are not aligned to their types");
    if (n >= MOST_ROWS)
        return fail(MF_E_UNSUPPORTED, "4-bit product of %lld rows", (long long)n);
    a.x = x, a.n = n, a.ldx = ldx, a.bias = bias, a.out = out;
    const HeldPlan plan(type, n, k, o, group, rows_in_pieces(x, ldx, type));
    if (bytes < plan.bytes || (plan.bytes && (!workspace || !aligned(workspace, 16))))
        return fail(MF_E_INVALID, "4-bit product's workspace of %lld bytes", (long long)bytes);
    return with_types(type, scale_type, [&](auto t, auto scale) {
        return launch_held<decltype(t), decltype(scale)>(a, plan, workspace, static_cast<hipStream_t>(stream));
    });
}

}  // extern "C"
