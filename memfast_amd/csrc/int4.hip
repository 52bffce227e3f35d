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

#include "mf_float.h"

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
    bool vec;               // rows of x are whole 16-byte pieces
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

// Eight values of a row from k on, zeros past the row's end.
template <typename T> struct alignas(16) Eight {
    T v[8];
    __device__ __forceinline__ void load(const T *row, i64 k, i64 end, bool vec) {
        if (vec && k + 8 <= end) {
#pragma unroll
            for (int i = 0; i < 8; i += PIECE<T>)
                *reinterpret_cast<Piece<T> *>(v + i) = *reinterpret_cast<const Piece<T> *>(row + k + i);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = k + i < end ? row[k + i] : T(0.0f);
        }
    }
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

// The four values that the quarters of a wave hold, each in all of them.
__device__ __forceinline__ void quarters(u32 v, u32 (&all)[4]) {
    const auto halves = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    const auto low = __builtin_amdgcn_permlane16_swap(halves[0], halves[0], false, false);
    const auto high = __builtin_amdgcn_permlane16_swap(halves[1], halves[1], false, false);
    all[0] = low[0], all[1] = low[1], all[2] = high[0], all[3] = high[1];
}

// ---- few rows --------------------------------------------------------------
// A workgroup takes OT tiles of outputs and all rows, its waves split the spans and add their sums in LDS in
// the order of the waves.  Row 4 i + quarter of a block of 16 rows is row 4 quarter + i of the matrix
// instruction, so that up to 4 rows need one register of its result and one scaling.
constexpr int FEW_WAVES = 8;

template <typename T, typename S, int OT, int NB, int R>
__global__ __launch_bounds__(64 * FEW_WAVES) void k_int4_few(const HeldArgs a) {
    typedef Operand<T> Op;
    constexpr int TERMS = Op::TERMS;
    extern __shared__ __align__(16) float sums[];   // [FEW_WAVES][OT * NB * R][64]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, quarter = lane >> 4, r = lane & 15;
    const i64 tiles = (a.o + TILE - 1) / TILE, tile0 = i64(blockIdx.x) * OT;
    const T *rows[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const i64 n = min(i64(16 * b + (r & 3) * 4 + (r >> 2)), a.n - 1);
        rows[b] = static_cast<const T *>(a.x) + n * a.ldx;
    }
    const u8 *codes[OT];
    const S *scales[OT];
    const u8 *zeros[OT];
#pragma unroll
    for (int t = 0; t < OT; ++t) {
        const i64 tile = min(tile0 + t, tiles - 1);
        codes[t] = a.codes + tile * a.spans * SPAN_BYTES + lane * 16;
        scales[t] = static_cast<const S *>(a.scales) + tile * a.groups * 16 + r;
        zeros[t] = a.zeros ? a.zeros + tile * a.groups * 16 + r : nullptr;
    }
    // Groups in a span: 4, 2 or 1; a quarter reads one of them.
    const int per = a.shift >= 7 ? 1 : 128 >> a.shift, group_steps = 4 / per;

    v4f total[OT][NB];
#pragma unroll
    for (int t = 0; t < OT; ++t)
#pragma unroll
        for (int b = 0; b < NB; ++b) total[t][b] = v4f{0, 0, 0, 0};

    v4u w[OT], next[OT];
    S s[OT], next_s[OT];
    u8 z[OT], next_z[OT];
    const auto fetch = [&](i64 span, v4u (&w)[OT], S (&s)[OT], u8 (&z)[OT]) {
        const i64 g = min((span * SPAN_K >> a.shift) + (quarter & (per - 1)), a.groups - 1) * 16;
#pragma unroll
        for (int t = 0; t < OT; ++t) {
            w[t] = *reinterpret_cast<const v4u *>(codes[t] + span * SPAN_BYTES);
            s[t] = scales[t][g];
            z[t] = zeros[t] ? zeros[t][g] : u8(8);
        }
    };
    if (wave < a.spans) fetch(wave, next, next_s, next_z);
    for (i64 span = wave; span < a.spans; span += FEW_WAVES) {
#pragma unroll
        for (int t = 0; t < OT; ++t) w[t] = next[t], s[t] = next_s[t], z[t] = next_z[t];
        if (span + FEW_WAVES < a.spans) fetch(span + FEW_WAVES, next, next_s, next_z);
        u32 scale[OT][4], zero[OT][4];
#pragma unroll
        for (int t = 0; t < OT; ++t) {
            quarters(__float_as_uint(float(s[t])), scale[t]);
            quarters(__float_as_uint(float(z[t])), zero[t]);
        }
        v4f acc[OT][NB], sum[NB];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            typename Op::V x[NB][TERMS], q[OT];
            const i64 k = span * SPAN_K + 32 * j + 8 * quarter;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                Eight<T> v;
                v.load(rows[b], k, a.k, a.vec);
                v.template split<TERMS>(x[b]);
            }
#pragma unroll
            for (int t = 0; t < OT; ++t) q[t] = Op::codes(w[t][j]);
            const bool begins = j % group_steps == 0, ends = (j + 1) % group_steps == 0;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                sum[b] = begins ? v4f{0, 0, 0, 0} : sum[b];
#pragma unroll
                for (int m = 0; m < TERMS; ++m) sum[b] = Op::mfma(x[b][m], Op::ones(), sum[b]);
#pragma unroll
                for (int t = 0; t < OT; ++t) {
                    acc[t][b] = begins ? v4f{0, 0, 0, 0} : acc[t][b];
#pragma unroll
                    for (int m = 0; m < TERMS; ++m) acc[t][b] = Op::mfma(x[b][m], q[t], acc[t][b]);
                }
            }
            if (ends) {
                const int g = j / group_steps;
#pragma unroll
                for (int t = 0; t < OT; ++t) {
                    const float sc = __uint_as_float(g == 0 ? scale[t][0] : g == 1 ? scale[t][1]
                                                     : g == 2 ? scale[t][2] : scale[t][3]);
                    const float ze = __uint_as_float(g == 0 ? zero[t][0] : g == 1 ? zero[t][1]
                                                     : g == 2 ? zero[t][2] : zero[t][3]);
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int i = 0; i < R; ++i)
                            total[t][b][i] = fmaf(sc, fmaf(-ze, sum[b][i], acc[t][b][i]), total[t][b][i]);
                }
            }
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
    for (int v = wave; v < VALUES; v += FEW_WAVES) {
        const int t = v / (NB * R), b = v / R % NB, i = v % R;
        const i64 n = 16 * b + 4 * i + quarter, o = (tile0 + t) * TILE + r;
        float y = 0.0f;
#pragma unroll
        for (int u = 0; u < FEW_WAVES; ++u) y += sums[(u * VALUES + v) * 64 + lane];
        if (n < a.n && o < a.o) {
            if (a.bias) y += float(static_cast<const T *>(a.bias)[o]);
            static_cast<T *>(a.out)[n * a.o + o] = rounded<T>(y);
        }
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

// One wave takes a group of one output: its peak, the scale peak / 7 in the scales' type, and the codes
// round(w / scale) + 8.  The bytes of codes are joined by the lanes of their two inputs.
template <typename T, typename S>
__global__ __launch_bounds__(256) void k_int4_quantize(const Int4QuantizeArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const i64 all = (a.o + TILE - 1) / TILE * TILE * a.groups;
    for (i64 id = i64(blockIdx.x) * 4 + wave; id < all; id += i64(gridDim.x) * 4) {
        const i64 o = id / a.groups, g = id - o * a.groups;
        const i64 first = g << a.shift, last = min(first + (i64(1) << a.shift), a.k);
        const T *w = static_cast<const T *>(a.w) + o * a.ldw;
        float peak = 0.0f;
        bool bad = false;
        if (o < a.o)
            for (i64 k = first + lane; k < last; k += 64) {
                const float v = fabsf(float(w[k]));
                bad |= !(v <= FLT_MAX);
                peak = fmaxf(peak, v);
            }
#pragma unroll
        for (int d = 32; d; d >>= 1) {
            peak = fmaxf(peak, __shfl_xor(peak, d));
            bad |= __shfl_xor(int(bad), d) != 0;
        }
        S held = S(peak > 0.0f ? peak / 7.0f : 1.0f);
        if (peak > 0.0f && !(float(held) > 0.0f)) held = S(1.0f);     // beneath the type: codes of 0
        if (bad) held = S(NAN);
        const float scale = float(held);
        if (lane == 0) static_cast<S *>(a.scales)[(o / TILE * a.groups + g) * 16 + o % TILE] = o < a.o ? held : S(0.0f);
        // Bytes hold inputs k and k + 4 of eight; zero codes' bytes past the last input are 8 twice.
        const i64 end = g + 1 == a.groups ? a.spans * SPAN_K : last;
        for (i64 p = (first >> 1) + lane; p < end >> 1; p += 64) {
            const i64 k = (p >> 2) * 8 + (p & 3);
            u32 byte = 0;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float c = 0.0f;
                if (o < a.o && k + 4 * i < last && !bad) c = rintf(float(w[k + 4 * i]) / scale);
                c = fminf(fmaxf(c, -8.0f), 7.0f);
                byte |= u32(int(c) + 8) << (4 * i);
            }
            const i64 in = k & (SPAN_K - 1);
            a.codes[((o / TILE) * a.spans + (k >> 7)) * SPAN_BYTES + (in >> 3 & 3) * 256 + o % TILE * 16 +
                    (in >> 5) * 4 + (in & 3)] = u8(byte);
        }
    }
}

// One lane restores one value.
template <typename T, typename S>
__global__ __launch_bounds__(256) void k_int4_dequantize(const HeldArgs a) {
    const i64 all = a.o * a.k;
    for (i64 id = i64(blockIdx.x) * 256 + threadIdx.x; id < all; id += i64(gridDim.x) * 256) {
        const i64 o = id / a.k, k = id - o * a.k, in = k & (SPAN_K - 1);
        const u32 byte = a.codes[((o / TILE) * a.spans + (k >> 7)) * SPAN_BYTES + (in >> 3 & 3) * 256 +
                                 o % TILE * 16 + (in >> 5) * 4 + (in & 3)];
        const i64 g = (o / TILE * a.groups + (k >> a.shift)) * 16 + o % TILE;
        const float zero = a.zeros ? float(a.zeros[g]) : 8.0f;
        const float q = float(byte >> (in & 4) & 15u);
        static_cast<T *>(a.out)[id] = T(float(static_cast<const S *>(a.scales)[g]) * (q - zero));
    }
}

// log2 of a group that is a power of two of at least 32, or -1.
int group_shift(i64 group) {
    for (int s = 5; s <= 24; ++s)
        if (group == i64(1) << s) return s;
    return -1;
}

constexpr i64 MOST_OUTPUTS = i64(1) << 27, MOST_INPUTS = i64(1) << 24;

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
    const i64 tiles = (a.o + TILE - 1) / TILE;
    const int lds = FEW_WAVES * OT * NB * R * 64 * int(sizeof(float));
    const auto kernel = k_int4_few<T, S, OT, NB, R>;
    const int status = allow_lds(kernel, lds);
    if (status) return status;
    hipLaunchKernelGGL(kernel, dim3(u32((tiles + OT - 1) / OT)), dim3(64 * FEW_WAVES), lds, s, a);
    return check_launch("4-bit product");
}

template <typename T, typename S> int launch_held(HeldArgs a, hipStream_t s) {
    // Blocks of up to 64 rows one after the other.
    const char *x = static_cast<const char *>(a.x);
    char *out = static_cast<char *>(a.out);
    for (i64 first = 0, n = a.n; first < n; first += 64) {
        a.x = x + first * a.ldx * i64(sizeof(T));
        a.out = out + first * a.o * i64(sizeof(T));
        a.n = std::min<i64>(64, n - first);
        const int status = a.n <= 4    ? launch_few<T, S, 2, 1, 1>(a, s)
                           : a.n <= 8  ? launch_few<T, S, 2, 1, 2>(a, s)
                           : a.n <= 16 ? launch_few<T, S, 2, 1, 4>(a, s)
                           : a.n <= 32 ? launch_few<T, S, 2, 2, 4>(a, s)
                           : a.n <= 48 ? launch_few<T, S, 2, 3, 4>(a, s)
                                       : launch_few<T, S, 2, 4, 4>(a, s);
        if (status) return status;
    }
    return MF_OK;
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
    if (!w || !known_type(type) || ldw < k || !aligned(w, type_bytes(type)))
        return fail(MF_E_INVALID, "invalid 4-bit quantization arguments");
    const Int4QuantizeArgs a{w, o, k, ldw, h.groups, h.spans, h.shift, codes, scales};
    const i64 units = (o + TILE - 1) / TILE * TILE * h.groups;
    const u32 grid = u32(std::min<i64>((units + 3) / 4, i64(1) << 20));
    return with_types(type, scale_type, [&](auto x, auto scale) {
        hipLaunchKernelGGL((k_int4_quantize<decltype(x), decltype(scale)>), dim3(grid), dim3(256), 0,
                           static_cast<hipStream_t>(stream), a);
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
    const u32 grid = u32(std::min<i64>((o * k + 255) / 256, i64(1) << 20));
    return with_type(type, [&](auto x) {
        return with_type(scale_type, [&](auto scale) {
            hipLaunchKernelGGL((k_int4_dequantize<decltype(x), decltype(scale)>), dim3(grid), dim3(256), 0,
                               static_cast<hipStream_t>(stream), a);
            return check_launch("4-bit dequantization");
        });
    });
}

int mf_int4_linear(const void *x, int32_t type, int64_t n, int64_t k, int64_t ldx, const uint8_t *codes,
                   const void *scales, int32_t scale_type, const uint8_t *zeros, int64_t o, int64_t group,
                   const void *bias, void *out, void *stream) {
    HeldArgs a{};
    const int status = check_held(codes, scales, scale_type, zeros, o, k, group, a);
    if (status) return status;
    if (!x || !known_type(type) || n < 1 || ldx < k || !out) 
        return fail(MF_E_INVALID, "invalid 4-bit product arguments");
    const uintptr_t one = type_bytes(type);
    if (!aligned(x, one) || !aligned(bias, one) || !aligned(out, one))
        return fail(MF_E_INVALID, "4-bit product's operands are not aligned to their types");
    if (n >= MOST_OUTPUTS)
        return fail(MF_E_UNSUPPORTED, "4-bit product of %lld rows", (long long)n);
    a.x = x, a.n = n, a.ldx = ldx, a.bias = bias, a.out = out;
    a.vec = aligned(x, 16) && ldx * i64(one) % 16 == 0;
    return with_types(type, scale_type, [&](auto t, auto scale) {
        return launch_held<decltype(t), decltype(scale)>(a, static_cast<hipStream_t>(stream));
    });
}

}  // extern "C"
