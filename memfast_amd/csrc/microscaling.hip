// 4-bit microscaled floating point: quantization and the product of two such operands.
//
// y = Q(x) Q(W)^T + b runs on v_mfma_scale_f32_*_f8f6f4, which takes one block of a row (16 bytes)
// and its scale byte per lane, so both operands go from memory to the matrix cores as they are.
// Sums are FP32.
#include <algorithm>
#include <type_traits>

#include "mf_mx.h"

namespace mf {

// ---------------------------------------------------------------------------
// Quantization
// ---------------------------------------------------------------------------
struct QuantizeJob {
    Job job;
    const void *x;      // [n, k], rows ldx apart
    i64 n, ldx;
    bool vec;
    u8 *codes, *scales;
    i64 row, seg;       // strides of the scales
};

// One launch quantizes up to two operands of one k and lays out a held operand's scales by segments.
struct QuantizeArgs {
    QuantizeJob q[2];
    i64 k;
    Job turn;
    const u8 *by_row;
    u8 *by_segment;
    i64 rows;
};

// One lane quantizes eight values and four neighbours share a block, so that every access is 16 bytes or
// whole lines. Bound by its bytes: 11008 x 4096 FP32 in 46 us, 204 MB at 4.4 TB/s (a copy: 5.0).
template <typename T>
__global__ __launch_bounds__(256) void k_mx_quantize(const QuantizeArgs a) {
    const i64 segs = segments(a.k);
    if (a.turn.mine(blockIdx.x)) {
        const i64 s = a.turn.unit();
        if (s < segs)
            for (i64 r = a.turn.row(); r < a.rows; r += a.turn.step())
                *reinterpret_cast<v2u *>(a.by_segment + (s * even(a.rows) + r) * SEG_SCALES) =
                    *reinterpret_cast<const v2u *>(a.by_row + (r * segs + s) * SEG_SCALES);
        return;
    }
    const QuantizeJob &q = a.q[a.q[1].job.mine(blockIdx.x) ? 1 : 0];
    const i64 unit = q.job.unit();
    if (unit >= segs * 32) return;
    const T *x = static_cast<const T *>(q.x);
    for (i64 r = q.job.row(); r < q.n; r += q.job.step()) {
        float v[8];
        load8(x + r * q.ldx, unit * 8, a.k, q.vec, v);
        u32 peak = peak8(v);
        peak = max(peak, u32(__shfl_xor(int(peak), 1)));
        peak = max(peak, u32(__shfl_xor(int(peak), 2)));
        const u32 byte = scale_byte(peak);
        reinterpret_cast<u32 *>(q.codes + r * segs * SEG_BYTES)[unit] = codes8(v, byte);
        if ((unit & 3) == 0)
            q.scales[r * q.row + unit / 32 * q.seg + (unit / 4 & 7)] = u8(byte);
    }
}

// One lane restores eight values. Bound by its bytes: 11008 x 4096 FP32 in 33 us, 204 MB.
template <typename T>
__global__ __launch_bounds__(256) void k_mx_dequantize(const Job job, const u8 *codes, const u8 *scales,
                                                       i64 n, i64 k, bool vec, T *out) {
    const i64 segs = segments(k), unit = job.unit();
    if (unit * 8 >= k) return;
    for (i64 r = job.row(); r < n; r += job.step()) {
        const v8bf exact = expand8(reinterpret_cast<const u32 *>(codes + r * segs * SEG_BYTES)[unit],
                                   scales[r * segs * SEG_SCALES + unit / 4]);
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = float(exact[i]);
        store8(out + r * k, unit * 8, k, vec, v);
    }
}

// ---------------------------------------------------------------------------
// Product
// ---------------------------------------------------------------------------
struct MxArgs {
    const u8 *xc, *wc;      // codes [n, segs * 128], [o, segs * 128]
    Scales xs, ws;
    const void *x;          // k_mx_few<..., true>: the input itself, rows ldx apart
    i64 ldx, k;
    bool vec;
    const void *bias;       // [o] or nullptr
    void *out;              // [n, o]
    i64 n, o, segs;
};

// ---- few rows --------------------------------------------------------------
// Few rows of x: the weight's bytes bound it, so each is loaded once, straight into the operand
// registers. A workgroup takes 16 rows of W; its eight waves split the segments and add their
// sums in LDS in the order of the waves. QUANTIZE: the workgroup quantizes x into LDS itself, while
// its first weights are on their way, which saves a launch; else Q(x) is read from the cache. Where W
// is not much larger, a wave's chain of two or three segments, its launch and the sums bound it: 1 x 4096 x
// 11008 BF16 7.7 us (24 MB of weight, 3.1 TB/s). With more rows it is also what every workgroup reads of Q(x):
// 24 x 11008 x 4096 10.5 us, 36 MB of x from the caches beside 24 MB of W; 64 rows 17 us, 96 MB of it.
constexpr int FEW_WAVES = 8, FEW_TILE = 16, AHEAD = 2;

__device__ __forceinline__ v4f mfma_few(v4u a, v4u b, v4f c, u32 sa, u32 sb) {
    const v8i av = {int(a.x), int(a.y), int(a.z), int(a.w), 0, 0, 0, 0};
    const v8i bv = {int(b.x), int(b.y), int(b.z), int(b.w), 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 0, int(sa), 0, int(sb));
}

// Rows of codes in LDS are 16 bytes apart from whole lines, so that 16 rows are in different banks.
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
    const u8 *wc = a.wc + o * a.segs * SEG_BYTES + block * 16, *ws = a.ws.data + o * a.ws.row;

    // AHEAD segments of the weight are under way: a compute unit's waves then keep more bytes in flight
    // for the memory's latency.
    v4u w[AHEAD][2];
    v2u sw[AHEAD];
    auto load_weight = [&](int slot, i64 s) {
        if (s < last) {
            w[slot][0] = *reinterpret_cast<const v4u *>(wc + s * SEG_BYTES);
            w[slot][1] = *reinterpret_cast<const v4u *>(wc + s * SEG_BYTES + 64);
            sw[slot] = *reinterpret_cast<const v2u *>(ws + s * a.ws.seg);
        }
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) load_weight(i, first + i);

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
    auto multiply = [&](int slot, i64 s) {
        v4u x0[NT], x1[NT];
        v2u sx[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const i64 r = min(i64(16 * t + row), a.n - 1);
            const u8 *xc = QUANTIZE ? staged + r * pitch : a.xc + r * a.segs * SEG_BYTES;
            const u8 *xs = QUANTIZE ? staged_scales + (r * a.segs + s) * SEG_SCALES
                                    : a.xs.data + r * a.xs.row + s * a.xs.seg;
            x0[t] = *reinterpret_cast<const v4u *>(xc + s * SEG_BYTES + block * 16);
            x1[t] = *reinterpret_cast<const v4u *>(xc + s * SEG_BYTES + 64 + block * 16);
            sx[t] = *reinterpret_cast<const v2u *>(xs);
        }
        const v4u w0 = w[slot][0], w1 = w[slot][1];
        const u32 sw0 = sw[slot].x >> (8 * block), sw1 = sw[slot].y >> (8 * block);
        load_weight(slot, s + AHEAD);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            acc[t] = mfma_few(x0[t], w0, acc[t], sx[t].x >> (8 * block), sw0);
            acc[t] = mfma_few(x1[t], w1, acc[t], sx[t].y >> (8 * block), sw1);
        }
    };
    for (i64 s = first; s < last; s += AHEAD)
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (s + i < last) multiply(i, s + i);
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

// WN x WO waves of TN x TO tiles of 32 x 32. A stage is one segment of every row of the tile (128 bytes of
// codes and 8 of scales), copied to LDS without passing through registers, STAGES - 1 stages ahead of
// the matrix cores. The 16-byte pieces of row r lie at p ^ (r / 2 & 7): the sixteen rows that a read serves
// at once, two to the 256 bytes of the banks, are then in different ones (p ^ (r & 7) has pairs of them
// meet: 78 against 70 us at 2048 x 4096 x 11008). That is 2640 TFLOP/s, above the 1150 to 1280 of a
// BF16 product; the matrix cores are busy 38% of the time, and the rest is the waves' wait for a stage's
// copies and each other (the reads of LDS take 24%, without conflicts).
template <typename T, int WN, int WO, int TN, int TO, int STAGES>
__global__ __launch_bounds__(64 * WN * WO) void k_mx_tile(const MxArgs a) {
    constexpr int BN = 32 * WN * TN, BO = 32 * WO * TO, ROWS = BN + BO, WAVES = WN * WO;
    constexpr int COPIES = ROWS / 8 / WAVES;                // of 8 rows' codes, by each wave
    constexpr int SCALE_COPIES = ROWS * SEG_SCALES / 1024;  // of 128 rows' scales, by as many waves
    constexpr int STAGE = ROWS * (SEG_BYTES + SEG_SCALES);
    static_assert(ROWS % (8 * WAVES) == 0 && ROWS % 128 == 0 && SCALE_COPIES <= WAVES, "whole copies");
    extern __shared__ __align__(16) u8 staged[];            // [STAGES][codes, scales]
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
        offset[i] = u32(at * pitch) + u32(((lane ^ r >> 1) & 7) * 16);
    }
    // Two rows' scales a lane; the even pitch of a segment holds the second of the last pair.
    const bool copies_scales = __builtin_amdgcn_readfirstlane(wave) < SCALE_COPIES;
    const int pair = (wave * 64 + lane) * 2;
    const u8 *scale_source = pair < BN ? a.xs.data + min(n0 + pair, even(a.n) - 2) * SEG_SCALES
                                       : a.ws.data + min(o0 + pair - BN, even(a.o) - 2) * SEG_SCALES;
    const i64 scale_step = pair < BN ? a.xs.seg : a.ws.seg;

    const u32 lds = lds_address(staged);
    auto copy = [&](i64 s, int buffer) {
        const u32 to = lds + buffer * STAGE;
#pragma unroll
        for (int i = 0; i < COPIES; ++i) {
            const int r = (first_copy + i) * 8;
            lds_dma_16((r < BN ? x0 : w0) + s * SEG_BYTES + offset[i],
                       __builtin_amdgcn_readfirstlane(to + r * SEG_BYTES));
        }
        if (copies_scales)
            lds_dma_16(scale_source + s * scale_step,
                       __builtin_amdgcn_readfirstlane(to + ROWS * SEG_BYTES + wave * 1024));
    };

    const int wn = (wave / WO) * TN * 32 + row, wo = BN + (wave % WO) * TO * 32 + row;
    v16f acc[TN][TO] = {};
    int filling = 0;            // the buffer of the next copy
    i64 next = 0;               // its segment
    for (; next < STAGES - 1 && next < a.segs; ++next) copy(next, filling++);
    int reading = 0;
    for (i64 s = 0; s < a.segs; ++s) {
        // All copies but those of the STAGES - 2 stages behind this one have to be there; near the
        // end there are fewer behind.
        if (s + STAGES - 2 < a.segs) {
            if (copies_scales)
                wait_stage<(STAGES - 2) * (COPIES + 1)>();
            else
                wait_stage<(STAGES - 2) * COPIES>();
        } else {
            wait_stage<0>();
        }
        if (next < a.segs) {
            copy(next++, filling);
            filling = filling + 1 == STAGES ? 0 : filling + 1;
        }
        const u8 *tile = staged + reading * STAGE, *scales = tile + ROWS * SEG_BYTES;
        reading = reading + 1 == STAGES ? 0 : reading + 1;
        u32 sx[TN], sw[TO];
#pragma unroll
        for (int i = 0; i < TN; ++i)
            sx[i] = half_scales(
                *reinterpret_cast<const v2u *>(scales + (wn + 32 * i) * SEG_SCALES), half);
#pragma unroll
        for (int j = 0; j < TO; ++j)
            sw[j] = half_scales(
                *reinterpret_cast<const v2u *>(scales + (wo + 32 * j) * SEG_SCALES), half);
        auto step = [&](auto number) {
            constexpr int STEP = decltype(number)::value;
            const int piece = ((2 * STEP + half) ^ (row >> 1 & 7)) * 16;
            v4u fx[TN], fw[TO];
#pragma unroll
            for (int i = 0; i < TN; ++i)
                fx[i] = *reinterpret_cast<const v4u *>(tile + (wn + 32 * i) * SEG_BYTES + piece);
#pragma unroll
            for (int j = 0; j < TO; ++j)
                fw[j] = *reinterpret_cast<const v4u *>(tile + (wo + 32 * j) * SEG_BYTES + piece);
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
    }
    T *out = static_cast<T *>(a.out);
#pragma unroll
    for (int j = 0; j < TO; ++j) {
        const i64 c = o0 + wo - BN + 32 * j;
        if (c >= a.o) continue;
        const float bias = a.bias ? float(static_cast<const T *>(a.bias)[c]) : 0.0f;
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const i64 r = n0 + wn - row + 32 * i + 8 * (e / 4) + 4 * half + (e & 3);
                if (r < a.n) out[r * a.o + c] = T(acc[i][j][e] + bias);
            }
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// Rows and columns whose scale offsets stay in 32 bits, and depths whose tiles' code offsets do.
static bool sizes_ok(i64 n, i64 k) { return n >= 1 && k >= 1 && n < i64(1) << 28 && k < i64(1) << 24; }

static bool operand_ok(const void *x, i64 n, i64 k, i64 ldx, const u8 *codes, const u8 *scales) {
    return x && codes && scales && sizes_ok(n, k) && (n == 1 || ldx >= k) && aligned(codes, 16) &&
           aligned(scales, 16);
}

template <typename T>
static QuantizeJob quantize_job(const void *x, i64 n, i64 k, i64 ldx, u8 *codes, Scales scales,
                                u32 &blocks) {
    return {add_job(segments(k) * 32, n, blocks),
            x, n, ldx, aligned(x, 16) && (n == 1 || ldx % PIECE<T> == 0),
            codes, const_cast<u8 *>(scales.data), scales.row, scales.seg};
}

struct ProductPlan {
    bool few;        // k_mx_few, else k_mx_tile
    bool quantize;   // Q(x) goes through memory
};

// k_mx_few reads Q(x) again for every 16 rows of W, k_mx_tile waits longer where it has few tiles (us, few
// / tiles, n x k x o; other widths were not timed, and the depth is not in the rule): 16 x 4096 x 11008 9.7
// / 9.3, 24 of them 12.0 / 9.4, 64 21.6 / 9.8; 24 x 11008 x 4096 10.3 / 18.9, 64 of them 16.9 / 19.2, 64 x
// 4096 x 4096 8.0 / 8.8.
constexpr i64 FEW_ROWS = 64, FEW_ROWS_WIDE = 16, WIDE = 8192;
// A launch has fewer than 2^32 threads; k_mx_few takes 32 an output.
constexpr i64 FEW_OUTPUTS = i64(1) << 26;
// Values of x that every workgroup may quantize again: 1 x 4096 x 11008 7.5 us against 8.1 and a launch of 3,
// 8 x 4096 x 11008 13.2 against 8.7 and 3.
constexpr i64 FEW_QUANTIZE = 16384;

static ProductPlan plan_product(i64 n, i64 k, i64 o, bool keep) {
    const bool few = n <= (o < WIDE ? FEW_ROWS : FEW_ROWS_WIDE) && o <= FEW_OUTPUTS;
    return {few, keep || !few || n > 16 || n * segments(k) * SEG > FEW_QUANTIZE};
}

template <typename T, int NT, bool QUANTIZE> static int launch_few_as(const MxArgs &args, hipStream_t s) {
    hipLaunchKernelGGL((k_mx_few<T, NT, QUANTIZE>), dim3(unsigned((args.o + FEW_TILE - 1) / FEW_TILE)),
                       dim3(64 * FEW_WAVES), QUANTIZE ? few_lds(args.n, args.segs) : 0, s, args);
    return check_launch("microscaled product");
}

template <typename T> static int launch_few(const MxArgs &args, const ProductPlan &plan, hipStream_t s) {
    if (!plan.quantize) return launch_few_as<T, 1, true>(args, s);
    if (args.n <= 16) return launch_few_as<T, 1, false>(args, s);
    return args.n <= 32 ? launch_few_as<T, 2, false>(args, s) : launch_few_as<T, 4, false>(args, s);
}

template <typename T, int WN, int WO, int TN, int TO, int STAGES>
static int launch_tile(const MxArgs &args, hipStream_t s) {
    constexpr int BN = 32 * WN * TN, BO = 32 * WO * TO;
    constexpr int LDS = STAGES * (BN + BO) * (SEG_BYTES + SEG_SCALES);
    const i64 tiles = (args.n + BN - 1) / BN * ((args.o + BO - 1) / BO);
    if (tiles > i64(1) << 30) return fail(MF_E_UNSUPPORTED, "product too large");
    auto kernel = k_mx_tile<T, WN, WO, TN, TO, STAGES>;
    if (const int status = allow_lds(kernel, LDS)) return status;
    hipLaunchKernelGGL(kernel, dim3(unsigned(tiles)), dim3(64 * WN * WO), LDS, s, args);
    return check_launch("microscaled product");
}

template <typename T> static int launch_tiles(const MxArgs &args, hipStream_t s) {
    // The largest tile of which every compute unit gets one (us, 64 x 64 / 128 x 128 / 128 x 256):
    // 2048 x 11008 x 4096 86 / 58 / 54, 777 x 1500 x 1111 5.7 / 9.2 / 11.0. A 256 x 256 tile is 1.14 times
    // as fast as two of 128 x 256 (43 against 49 us at 4096^3) where it does not leave more of the last
    // round empty (77 against 70 us at 2048 x 4096 x 11008). A third stage takes 128 x 256 from 54 to 55 us,
    // and 128 x 128 the second workgroup of a compute unit: from 60 to 74 us.
    const auto tiles = [&](i64 bn, i64 bo) { return (args.n + bn - 1) / bn * ((args.o + bo - 1) / bo); };
    const auto rounds = [&](i64 bn, i64 bo) { return (tiles(bn, bo) + 255) / 256; };
    if (tiles(128, 256) >= 256) {
        if (tiles(256, 256) >= 192 && rounds(256, 256) * 12 <= rounds(128, 256) * 7)
            return launch_tile<T, 2, 4, 4, 2, 2>(args, s);
        return launch_tile<T, 2, 4, 2, 2, 2>(args, s);
    }
    if (tiles(128, 128) >= 256) return launch_tile<T, 2, 2, 2, 2, 2>(args, s);
    // With a tile or less for each compute unit, more stages stand in for other workgroups: 64 x 4096 x
    // 11008 14.7 / 9.8 us with two / four.
    if (tiles(64, 64) <= 256) return launch_tile<T, 2, 2, 1, 1, 4>(args, s);
    return launch_tile<T, 2, 2, 1, 1, 2>(args, s);
}

}  // namespace mf

using namespace mf;

extern "C" {

int mf_mx_quantize(const void *x, int32_t type, int64_t n, int64_t k, int64_t ldx, uint8_t *codes,
                   uint8_t *scales, void *stream) {
    if (!known_type(type) || !operand_ok(x, n, k, ldx, codes, scales))
        return fail(MF_E_INVALID, "invalid microscaled quantization arguments");
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        QuantizeArgs args{};
        u32 blocks = 0;
        args.k = k;
        args.q[0] = quantize_job<T>(x, n, k, ldx, codes, scales_by_row(scales, segments(k)), blocks);
        hipLaunchKernelGGL(k_mx_quantize<T>, dim3(blocks), dim3(256), 0,
                           static_cast<hipStream_t>(stream), args);
        return check_launch("microscaled quantization");
    });
}

int mf_mx_dequantize(const uint8_t *codes, const uint8_t *scales, int64_t n, int64_t k, void *out,
                     int32_t type, void *stream) {
    if (!out || !known_type(type) || !operand_ok(out, n, k, k, codes, scales))
        return fail(MF_E_INVALID, "invalid microscaled dequantization arguments");
    u32 blocks = 0;
    const Job job = add_job((k + 7) / 8, n, blocks);
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        const bool vec = aligned(out, 16) && (n == 1 || k % PIECE<T> == 0);
        hipLaunchKernelGGL(k_mx_dequantize<T>, dim3(blocks), dim3(256), 0,
                           static_cast<hipStream_t>(stream), job, codes, scales, n, k, vec,
                           static_cast<T *>(out));
        return check_launch("microscaled dequantization");
    });
}

int mf_mx_linear_sizes(int64_t n, int64_t k, int64_t o, int32_t held, int32_t keep, int64_t *xcodes,
                       int64_t *workspace) {
    if (!xcodes || !workspace || !sizes_ok(n, k) || !sizes_ok(o, k))
        return fail(MF_E_INVALID, "invalid microscaled product sizes");
    const ProductPlan plan = plan_product(n, k, o, keep);
    *xcodes = plan.quantize ? n * segments(k) * SEG_BYTES : 0;
    *workspace = held && !plan.few ? even(o) * segments(k) * SEG_SCALES : 0;
    return MF_OK;
}

int mf_mx_linear(const void *x, int32_t type, int64_t n, int64_t k, int64_t ldx, const void *weight,
                 int64_t ldw, uint8_t *wcodes, uint8_t *wscales, int64_t o, const void *bias,
                 int32_t keep, uint8_t *xcodes, uint8_t *xscales, void *out, void *workspace,
                 int64_t bytes, void *stream) {
    if (!known_type(type) || !sizes_ok(n, k) || !out || !x || (n > 1 && ldx < k) ||
        !operand_ok(weight ? weight : wcodes, o, k, weight ? ldw : k, wcodes, wscales))
        return fail(MF_E_INVALID, "invalid microscaled product arguments");
    const ProductPlan plan = plan_product(n, k, o, keep);
    const i64 segs = segments(k);
    const bool turn = !weight && !plan.few;
    if (plan.quantize && !operand_ok(x, n, k, ldx, xcodes, xscales))
        return fail(MF_E_INVALID, "missing or unaligned codes or scales of a product");
    if (turn && (!workspace || bytes < even(o) * segs * SEG_SCALES || !aligned(workspace, 16)))
        return fail(MF_E_INVALID, "product workspace is missing, unaligned or too small");
    hipStream_t s = static_cast<hipStream_t>(stream);
    MxArgs args{};
    args.xc = xcodes;
    args.xs = scales_by_segment(xscales, n);
    args.wc = wcodes;
    args.ws = weight ? scales_by_segment(wscales, o)
                     : turn ? scales_by_segment(static_cast<const u8 *>(workspace), o)
                            : scales_by_row(wscales, segs);
    args.x = x;
    args.ldx = ldx;
    args.k = k;
    args.bias = bias;
    args.out = out;
    args.n = n;
    args.o = o;
    args.segs = segs;
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        QuantizeArgs q{};
        u32 blocks = 0;
        q.k = k;
        if (plan.quantize) q.q[0] = quantize_job<T>(x, n, k, ldx, xcodes, args.xs, blocks);
        if (weight) q.q[1] = quantize_job<T>(weight, o, k, ldw, wcodes, args.ws, blocks);
        if (turn) {
            q.turn = add_job(segs, o, blocks);
            q.by_row = wscales;
            q.by_segment = static_cast<u8 *>(workspace);
            q.rows = o;
        }
        if (blocks) {
            hipLaunchKernelGGL(k_mx_quantize<T>, dim3(blocks), dim3(256), 0, s, q);
            if (const int status = check_launch("microscaled quantization")) return status;
        }
        args.vec = aligned(x, 16) && (n == 1 || ldx % PIECE<T> == 0);
        return plan.few ? launch_few<T>(args, plan, s) : launch_tiles<T>(args, s);
    });
}

}  // extern "C"
