// Distillation from a teacher's top logits: the largest logits of each row with the mass of the
// others, and the loss of a student against them with its gradient.
//
// Teacher: p = softmax([v_1 / T, ..., v_k / T, tail]) over the entries that are present (index >= 0)
// and one bucket for every other class; without a tail that bucket is empty.
// Student: z = s / T, q = softmax(z) over the V classes, q_r the sum of q outside the entries.
//   loss = T^2 KL(p || q) = T^2 sum over entries and the bucket of p log(p / q).
//   dloss/ds_c = T (q_c - p_c) at an entry,  T q_c (1 - p_r / q_r) elsewhere.
// The loss is summed as p log(p / q) - p + q: the added q - p cancel over the buckets, and what
// is left are terms that are never negative, so that a student near its teacher keeps its digits.
//
// Exponentials are powers of two, exp2((x - m) c) with c = log2(e) / T and m the largest x: the
// difference comes first, so that logits of the type's lowest value, which masks use, stay finite.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "mf_float.h"

namespace mf {

constexpr float LOG2E = 1.44269504f, LN2 = 0.693147181f;
constexpr int MOST_ENTRIES = 1024;
constexpr i64 MOST_CLASSES = i64(1) << 20;   // one bit each in LDS: 128 KiB

__device__ __forceinline__ float power(float x, float m, float c) {
    return __builtin_amdgcn_exp2f((x - m) * c);
}

// A maximum m and the sum of exp2((x - m) c); m = -inf and 0 for nothing at all.
struct LogSum {
    float m = -INFINITY, s = 0.0f;
    // What values are subtracted from: a maximum of -inf stands for values that are all -inf.
    __device__ __forceinline__ float ref() const { return m == -INFINITY ? 0.0f : m; }
    __device__ __forceinline__ void merge(float m2, float s2, float c) {
        const float old = m;
        m = fmaxf(m, m2);
        s = s * power(old, ref(), c) + s2 * power(m2, ref(), c);
    }
    __device__ __forceinline__ void add(float x, float c) {
        merge(x, x == -INFINITY ? 0.0f : 1.0f, c);
    }
};

// Over a workgroup; every thread gets the result. `scratch` holds two floats a wave.
template <int WAVES> __device__ LogSum block_merge(LogSum v, float c, float *scratch) {
    for (int d = 32; d; d >>= 1) v.merge(__shfl_xor(v.m, d), __shfl_xor(v.s, d), c);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        scratch[2 * (threadIdx.x >> 6)] = v.m;
        scratch[2 * (threadIdx.x >> 6) + 1] = v.s;
    }
    __syncthreads();
    LogSum all;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) all.merge(scratch[2 * w], scratch[2 * w + 1], c);
    return all;
}

template <int WAVES> __device__ float block_sum(float v, float *scratch) {
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    float all = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) all += scratch[w];
    return all;
}

// A row in 16-byte pieces at 16-byte addresses: piece i holds the classes i * P - off to
// i * P - off + P - 1, the first and last pieces fewer where the row starts or ends inside them.
template <typename T> struct Row {
    const T *data;
    i64 v;
    int off;
    i64 pieces;
    __device__ __forceinline__ Row(const T *p, i64 classes) : data(p), v(classes) {
        off = int(reinterpret_cast<uintptr_t>(p) % 16 / sizeof(T));
        pieces = (off + v + PIECE<T> - 1) / PIECE<T>;
    }
    __device__ __forceinline__ bool whole(i64 i) const {
        return i * PIECE<T> >= off && (i + 1) * PIECE<T> <= off + v;
    }
    // The piece's values, `fill` outside the row.
    __device__ __forceinline__ void load(i64 i, float fill, float (&x)[PIECE<T>]) const {
        const i64 first = i * PIECE<T> - off;
        if (whole(i)) {
            const Piece<T> piece = *reinterpret_cast<const Piece<T> *>(data + first);
#pragma unroll
            for (int j = 0; j < PIECE<T>; ++j) x[j] = float(piece.v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < PIECE<T>; ++j)
                x[j] = first + j >= 0 && first + j < v ? float(data[first + j]) : fill;
        }
    }
};

// One bit for each class, in the order of the row's pieces.
template <typename T>
__device__ __forceinline__ u32 piece_bits(const u32 *bits, i64 i) {
    constexpr int P = PIECE<T>;
    return bits[i * P / 32] >> (i * P % 32) & ((1u << P) - 1u);
}

struct DistillArgs {
    const void *logits;      // [n, ld]
    const void *values;      // [n, k] of values_type
    int values_type;
    const i64 *indices;      // [n, k]
    const float *tail;       // [n] or nullptr
    const float *weight;     // [n] or nullptr
    i64 n, v, ld, k;
    float temperature;
    float *row_loss;         // [n]
    float *ref, *coef;       // [n]: a class outside the entries has the gradient
                             // exp2((s - ref) c) * coef (times T, weight and the incoming one)
    float *entry_grad;       // [n, k]: q - p
};

// p d - p + q with d = log(p / q), as p (d + exp(-d) - 1) where that stays in range. d is formed
// and expanded in 64 bits: its terms cancel to the order of d^2, and there are k + 1 of them a row.
__device__ __forceinline__ float bucket_loss(float p, float q, double d) {
    if (p == 0.0f) return q;
    return d > -8.0 ? p * float(d + expm1(-d)) : p * float(d) + (q - p);
}

__device__ __forceinline__ float value_at(const void *values, int type, i64 i) {
    if (type == MF_F32) return static_cast<const float *>(values)[i];
    if (type == MF_BF16) return float(static_cast<const bf16 *>(values)[i]);
    return float(static_cast<const f16 *>(values)[i]);
}

// Marks the row's entries and returns whether any index is outside the row or repeated.
__device__ __forceinline__ bool mark_entries(const i64 *indices, i64 k, i64 v, int off, u32 *bits,
                                             i64 words, int threads) {
    for (i64 w = threadIdx.x; w < words; w += threads) bits[w] = 0;
    __syncthreads();
    bool bad = false;
    for (i64 j = threadIdx.x; j < k; j += threads) {
        const i64 index = indices[j];
        if (index < -1 || index >= v) {
            bad = true;
        } else if (index >= 0) {
            const u32 bit = 1u << ((index + off) & 31);
            bad = bad || (atomicOr(&bits[(index + off) >> 5], bit) & bit);
        }
    }
    return __syncthreads_or(bad);
}

// One workgroup a row: one pass over the row for the classes outside the entries.
template <typename T, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_distill(const DistillArgs a) {
    extern __shared__ u32 bits[];
    __shared__ float scratch[2 * WAVES];
    constexpr int THREADS = 64 * WAVES;
    const i64 r = blockIdx.x;
    const float weight = a.weight ? a.weight[r] : 1.0f;
    if (weight == 0.0f) {   // nothing of such a row is read
        for (i64 j = threadIdx.x; j < a.k; j += THREADS) a.entry_grad[r * a.k + j] = 0.0f;
        if (threadIdx.x == 0) a.row_loss[r] = a.ref[r] = a.coef[r] = 0.0f;
        return;
    }
    const T *s = static_cast<const T *>(a.logits) + r * a.ld;
    const i64 first = r * a.k;
    const i64 *indices = a.indices + r * a.k;
    const Row<T> row(s, a.v);
    const float c = LOG2E / a.temperature;
    const bool bad = mark_entries(indices, a.k, a.v, row.off, bits, (row.off + a.v + 31) / 32,
                                  THREADS);

    LogSum teacher, entries, rest;
    if (!bad)
        for (i64 j = threadIdx.x; j < a.k; j += THREADS)
            if (indices[j] >= 0) {
                teacher.add(value_at(a.values, a.values_type, first + j), c);
                entries.add(float(s[indices[j]]), c);
            }
    for (i64 i = threadIdx.x; i < row.pieces; i += THREADS) {
        float x[PIECE<T>];
        row.load(i, -INFINITY, x);
        const u32 marked = piece_bits<T>(bits, i);
        const float old = rest.m;
#pragma unroll
        for (int j = 0; j < PIECE<T>; ++j) {
            if (marked >> j & 1u) x[j] = -INFINITY;
            rest.m = fmaxf(rest.m, x[j]);
        }
        const float ref = rest.ref();
        rest.s *= power(old, ref, c);
#pragma unroll
        for (int j = 0; j < PIECE<T>; ++j) rest.s += power(x[j], ref, c);
    }
    teacher = block_merge<WAVES>(teacher, c, scratch);
    entries = block_merge<WAVES>(entries, c, scratch);
    rest = block_merge<WAVES>(rest, c, scratch);

    const float tail = a.tail ? a.tail[r] * a.temperature : -INFINITY;   // as a logit
    const bool empty = teacher.m == -INFINITY && teacher.s == 0.0f && tail == -INFINITY;
    teacher.add(tail, c);
    LogSum all = rest;
    all.merge(entries.m, entries.s, c);
    const float t0 = teacher.ref(), z0 = all.ref();
    // log(p / q) = ((t - t0) - (z - z0)) / T - shift.
    const double cold = 1.0 / double(a.temperature);
    const double shift = log(double(teacher.s)) - log(double(all.s));
    float loss = 0.0f;
    for (i64 j = threadIdx.x; j < a.k; j += THREADS) {
        float grad = 0.0f;
        if (bad) {
            grad = NAN;
        } else if (indices[j] >= 0 && !empty) {
            const float t = value_at(a.values, a.values_type, first + j);
            const float z = float(s[indices[j]]);
            const float p = power(t, t0, c) / teacher.s;
            const float q = power(z, z0, c) / all.s;
            loss += bucket_loss(p, q, ((double(t) - t0) - (double(z) - z0)) * cold - shift);
            grad = q - p;
        }
        a.entry_grad[r * a.k + j] = grad;
    }
    loss = block_sum<WAVES>(loss, scratch);
    if (threadIdx.x == 0) {
        float coef = 0.0f;
        if (bad) {
            loss = coef = NAN;
        } else if (!empty) {
            const float p = power(tail, t0, c) / teacher.s;
            const float scale = power(rest.ref(), z0, c) / all.s;
            const float q = rest.s * scale;
            const double student = (double(rest.ref()) - z0) * cold + log(double(rest.s));
            loss += bucket_loss(p, q, (double(tail) - t0) * cold - student - shift);
            // Without any finite class outside the entries there is nothing to scale.
            coef = rest.s == 0.0f ? (p > 0.0f ? NAN : 0.0f) : scale - p / rest.s;
        }
        a.row_loss[r] = loss * a.temperature * a.temperature;
        a.ref[r] = rest.ref();
        a.coef[r] = coef;
    }
}

// sum(weight * loss) over the rows, divided by sum(weight) where `mean`, in a fixed order, in FP64;
// norm = 1 / sum(weight) (0 where there is no weight) or 1.
__global__ __launch_bounds__(256) void k_distill_total(const float *row_loss, const float *weight, i64 n,
                                                       bool mean, float *loss, float *norm) {
    __shared__ double part[2][256];
    double sum = 0.0, weights = 0.0;
    for (i64 r = threadIdx.x; r < n; r += 256) {
        const float w = weight ? weight[r] : 1.0f;
        sum += double(w) * double(row_loss[r]);
        weights += w;
    }
    part[0][threadIdx.x] = sum;
    part[1][threadIdx.x] = weights;
    for (int d = 128; d; d >>= 1) {
        __syncthreads();
        if (int(threadIdx.x) < d) {
            part[0][threadIdx.x] += part[0][threadIdx.x + d];
            part[1][threadIdx.x] += part[1][threadIdx.x + d];
        }
    }
    if (threadIdx.x == 0) {
        const double total = part[1][0];
        const double scale = mean ? (total == 0.0 ? 0.0 : 1.0 / total) : 1.0;
        *loss = total == 0.0 && mean ? 0.0f : float(part[0][0] * scale);
        *norm = float(scale);
    }
}

struct DistillGradArgs {
    const void *logits;
    const i64 *indices;
    const float *weight, *ref, *coef, *entry_grad;
    const float *norm;        // nullptr: 1
    const float *incoming;    // incoming[r * incoming_step]
    i64 incoming_step;
    i64 n, v, ld, k;
    float temperature;
    void *grad;               // [n, v]
};

// Writes a piece of the gradient; entries are left to the threads that hold them.
template <typename T>
__device__ __forceinline__ void store_rest(T *grad, const Row<T> &row, i64 i, u32 marked,
                                           const float (&x)[PIECE<T>]) {
    const i64 first = i * PIECE<T> - row.off;
    const bool vec = (reinterpret_cast<uintptr_t>(grad + first) & 15) == 0;
    if (marked == 0 && vec && row.whole(i)) {
        Piece<T> piece;
#pragma unroll
        for (int j = 0; j < PIECE<T>; ++j) piece.v[j] = T(x[j]);
        *reinterpret_cast<Piece<T> *>(grad + first) = piece;
    } else {
#pragma unroll
        for (int j = 0; j < PIECE<T>; ++j)
            if (first + j >= 0 && first + j < row.v && !(marked >> j & 1u)) grad[first + j] = T(x[j]);
    }
}

template <typename T, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_distill_grad(const DistillGradArgs a) {
    extern __shared__ u32 bits[];
    constexpr int THREADS = 64 * WAVES;
    const i64 r = blockIdx.x;
    const Row<T> row(static_cast<const T *>(a.logits) + r * a.ld, a.v);
    T *grad = static_cast<T *>(a.grad) + r * a.v;
    const i64 *indices = a.indices + r * a.k;
    const float weight = a.weight ? a.weight[r] : 1.0f;
    const float scale = weight == 0.0f ? 0.0f
                                       : a.incoming[r * a.incoming_step] * weight *
                                             (a.norm ? *a.norm : 1.0f) * a.temperature;
    const float c = LOG2E / a.temperature, ref = a.ref[r], coef = a.coef[r] * scale;
    const bool bad = mark_entries(indices, a.k, a.v, row.off, bits, (row.off + a.v + 31) / 32,
                                  THREADS);
    for (i64 i = threadIdx.x; i < row.pieces; i += THREADS) {
        float x[PIECE<T>];
        if (coef == 0.0f) {   // nothing flows back, whatever the logits are
#pragma unroll
            for (int j = 0; j < PIECE<T>; ++j) x[j] = 0.0f;
        } else {
            row.load(i, 0.0f, x);
#pragma unroll
            for (int j = 0; j < PIECE<T>; ++j)
                x[j] = power(x[j], ref, c) * coef;
        }
        store_rest(grad, row, i, piece_bits<T>(bits, i), x);
    }
    for (i64 j = threadIdx.x; j < a.k; j += THREADS) {
        const i64 index = indices[j];
        if (index >= 0 && index < a.v) {
            const float g = a.entry_grad[r * a.k + j];
            grad[index] = T(bad && weight != 0.0f ? NAN : scale == 0.0f ? 0.0f : g * scale);
        }
    }
}

// ---------------------------------------------------------------------------
// The largest logits of a row
// ---------------------------------------------------------------------------
// A class's key: larger for a larger logit, and for the lower index among equal ones. NaN counts as
// the largest value; -0 equals 0.
__device__ __forceinline__ u32 order_of(float x) {
    const u32 u = __float_as_uint(x + 0.0f);
    if (x != x) return 0xffffffffu;
    return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ u64 key_of(float x, i64 index) {
    return u64(order_of(x)) << 32 | (0xffffffffu - u32(index));
}

struct TopArgs {
    const void *logits;   // [n, ld]
    i64 n, v, ld;
    int k;
    float temperature;
    void *values;         // [n, k]
    i64 *indices;         // [n, k]
    float *tail;          // [n]
};

// Radix selection of the k-th largest key, eight bits at a time, then the selected keys in order and
// the others' sum.
template <typename T, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_top_select(const TopArgs a) {
    __shared__ u64 list[MOST_ENTRIES];
    __shared__ u32 counts[256];
    __shared__ u32 digit, remaining, found, last;
    __shared__ float scratch[2 * WAVES];
    constexpr int THREADS = 64 * WAVES;
    const i64 r = blockIdx.x;
    const T *s = static_cast<const T *>(a.logits) + r * a.ld;
    const Row<T> row(s, a.v);
    u64 prefix = 0;
    if (threadIdx.x == 0) remaining = a.k;
    int shift = 56;
    for (;; shift -= 8) {
        __syncthreads();
        for (int b = threadIdx.x; b < 256; b += THREADS) counts[b] = 0;
        __syncthreads();
        for (i64 i = threadIdx.x; i < row.pieces; i += THREADS) {
            float x[PIECE<T>];
            row.load(i, 0.0f, x);
#pragma unroll
            for (int j = 0; j < PIECE<T>; ++j) {
                const i64 index = i * PIECE<T> - row.off + j;
                const u64 key = key_of(x[j], index);
                if (index >= 0 && index < a.v &&
                    (shift == 56 || key >> (shift + 8) == prefix >> (shift + 8)))
                    atomicAdd(&counts[key >> shift & 255u], 1u);
            }
        }
        __syncthreads();
        if (threadIdx.x == 0) {   // the digit that holds the k-th largest
            u32 left = remaining;
            int d = 255;
            while (counts[d] < left) left -= counts[d--];
            digit = d;
            remaining = left;
            last = counts[d] == left;
        }
        __syncthreads();
        prefix |= u64(digit) << shift;
        if (last || shift == 0) break;
    }
    // Every key from prefix on is selected: k of them.
    int pow2 = 1;
    while (pow2 < a.k) pow2 <<= 1;
    for (int j = threadIdx.x; j < pow2; j += THREADS) list[j] = 0;
    if (threadIdx.x == 0) found = 0;
    __syncthreads();
    const float c = LOG2E / a.temperature;
    LogSum rest;
    for (i64 i = threadIdx.x; i < row.pieces; i += THREADS) {
        float x[PIECE<T>];
        row.load(i, -INFINITY, x);
#pragma unroll
        for (int j = 0; j < PIECE<T>; ++j) {
            const i64 index = i * PIECE<T> - row.off + j;
            if (index < 0 || index >= a.v) continue;
            const u64 key = key_of(x[j], index);
            if (key >= prefix) {
                const u32 at = atomicAdd(&found, 1u);
                if (at < u32(a.k)) list[at] = key;
            } else {
                rest.add(x[j], c);
            }
        }
    }
    __syncthreads();
    for (int size = 2; size <= pow2; size <<= 1)
        for (int stride = size >> 1; stride; stride >>= 1) {
            for (int j = threadIdx.x; j < pow2; j += THREADS) {
                const int other = j ^ stride;
                if (other > j) {
                    const u64 x = list[j], y = list[other];
                    if ((x < y) == ((j & size) == 0)) {
                        list[j] = y;
                        list[other] = x;
                    }
                }
            }
            __syncthreads();
        }
    for (int j = threadIdx.x; j < a.k; j += THREADS) {
        const i64 index = i64(0xffffffffu - u32(list[j]));
        a.indices[r * a.k + j] = index;
        static_cast<T *>(a.values)[r * a.k + j] = s[index];
    }
    rest = block_merge<WAVES>(rest, c, scratch);
    if (threadIdx.x == 0)
        a.tail[r] = rest.m == -INFINITY && rest.s == 0.0f
                        ? -INFINITY
                        : rest.ref() / a.temperature + __builtin_amdgcn_logf(rest.s) * LN2;
}

static int check_rows(const char *what, const void *logits, int32_t type, i64 n, i64 v, i64 ld, i64 k,
                      float temperature) {
    if (!logits || !known_type(type) || n < 1 || v < 1 || k < 1 || k > v || (n > 1 && ld < v) ||
        !(temperature > 0.0f) || !(temperature <= FLT_MAX) || !aligned(logits, type_bytes(type)))
        return fail(MF_E_INVALID, "invalid %s arguments", what);
    if (v > MOST_CLASSES || n > i64(1) << 30)
        return fail(MF_E_UNSUPPORTED, "%s takes at most %lld classes", what, (long long)MOST_CLASSES);
    if (k > MOST_ENTRIES)
        return fail(MF_E_UNSUPPORTED, "%s takes at most %d entries a row", what, MOST_ENTRIES);
    return MF_OK;
}

constexpr int ROW_WAVES = 8;

static size_t mark_bytes(i64 v) { return size_t((v + 8 + 31) / 32 * 4); }

// Dynamic LDS above 64 KiB has to be asked for once per kernel and device.
template <typename K> static int allow_lds(K kernel, size_t bytes) {
    if (bytes <= 48 << 10) return MF_OK;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
    return e == hipSuccess ? MF_OK : fail(MF_E_RESOURCE, "LDS of %zu bytes: %s", bytes,
                                          hipGetErrorString(e));
}

}  // namespace mf

using namespace mf;

extern "C" {

int mf_top_logits(const void *logits, int32_t type, int64_t n, int64_t v, int64_t ld, int64_t k,
                  float temperature, void *values, int64_t *indices, float *tail, void *stream) {
    const int status = check_rows("top logits", logits, type, n, v, ld, k, temperature);
    if (status) return status;
    if (!values || !indices || !tail) return fail(MF_E_INVALID, "invalid top logits arguments");
    const TopArgs args{logits, n, v, ld, int(k), temperature, values, indices, tail};
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        hipLaunchKernelGGL((k_top_select<T, 16>), dim3(unsigned(n)), dim3(1024), 0,
                           static_cast<hipStream_t>(stream), args);
        return check_launch("top logits");
    });
}

int mf_distill_loss(const void *logits, int32_t type, int64_t n, int64_t v, int64_t ld,
                    const void *values, int32_t values_type, const int64_t *indices,
                    const float *tail, int64_t k, float temperature, const float *weight,
                    int32_t reduction, float *row_loss,
                    float *ref, float *coef, float *entry_grad, float *loss, float *norm,
                    void *stream) {
    const int status = check_rows("distillation", logits, type, n, v, ld, k, temperature);
    if (status) return status;
    if (!values || !known_type(values_type) || !indices || !row_loss || !ref || !coef || !entry_grad || reduction < 0 ||
        reduction > 2 || (reduction != MF_SUM_NONE && (!loss || !norm)))
        return fail(MF_E_INVALID, "invalid distillation arguments");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const DistillArgs args{logits, values, values_type, indices, tail, weight, n, v, ld, k,
                           temperature, row_loss, ref, coef, entry_grad};
    const int launched = with_type(type, [&](auto zero) {
        using T = decltype(zero);
        const int lds = allow_lds(k_distill<T, ROW_WAVES>, mark_bytes(v));
        if (lds) return lds;
        hipLaunchKernelGGL((k_distill<T, ROW_WAVES>), dim3(unsigned(n)), dim3(64 * ROW_WAVES),
                           mark_bytes(v), s, args);
        return check_launch("distillation loss");
    });
    if (launched || reduction == MF_SUM_NONE) return launched;
    hipLaunchKernelGGL(k_distill_total, dim3(1), dim3(256), 0, s, row_loss, weight, n,
                       reduction == MF_SUM_MEAN, loss, norm);
    return check_launch("distillation total");
}

int mf_distill_grad(const void *logits, int32_t type, int64_t n, int64_t v, int64_t ld,
                    const int64_t *indices, int64_t k, float temperature, const float *weight,
                    const float *ref, const float *coef, const float *entry_grad, const float *norm,
                    const float *incoming, int64_t incoming_step, void *grad, void *stream) {
    const int status = check_rows("distillation gradient", logits, type, n, v, ld, k, temperature);
    if (status) return status;
    if (!indices || !ref || !coef || !entry_grad || !incoming || !grad || incoming_step < 0)
        return fail(MF_E_INVALID, "invalid distillation gradient arguments");
    const DistillGradArgs args{logits, indices, weight, ref, coef, entry_grad, norm, incoming,
                               incoming_step, n, v, ld, k, temperature, grad};
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        const int lds = allow_lds(k_distill_grad<T, ROW_WAVES>, mark_bytes(v));
        if (lds) return lds;
        hipLaunchKernelGGL((k_distill_grad<T, ROW_WAVES>), dim3(unsigned(n)), dim3(64 * ROW_WAVES),
                           mark_bytes(v), static_cast<hipStream_t>(stream), args);
        return check_launch("distillation gradient");
    });
}

}  // extern "C"
