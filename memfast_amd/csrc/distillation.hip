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

template <int WAVES, typename V> __device__ V block_sum(V v, float *scratch) {
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    V *part = reinterpret_cast<V *>(scratch);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    V all = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) all += part[w];
    return all;
}

template <int WAVES> __device__ float block_max(float v, float *scratch) {
    for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    float all = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) all = fmaxf(all, scratch[w]);
    return all;
}

// A row in 16-byte pieces at 16-byte addresses: piece i holds the classes i * P - off to
// i * P - off + P - 1; pieces first to last - 1 are whole, and the one before or after them, where the row
// starts or ends inside one, is read class by class. A row has at most 2^20 classes.
template <typename T> struct Row {
    static constexpr int P = PIECE<T>;
    const T *data;
    int v, off, pieces, first, last;
    __device__ __forceinline__ Row(const T *p, i64 classes) : data(p), v(int(classes)) {
        off = int(reinterpret_cast<uintptr_t>(p) % 16 / sizeof(T));
        pieces = (off + v + P - 1) / P;
        first = off ? 1 : 0;
        last = (off + v) / P;
    }
    // A whole piece, at one 32-bit offset from the row's address. ONCE: it is not read again, and a
    // non-temporal load leaves the cache to others (one pass over 2048 x 128000 BF16 118 -> 110 us).
    template <bool ONCE> __device__ __forceinline__ v4u whole(int i) const {
        const v4u *p = reinterpret_cast<const v4u *>(reinterpret_cast<const char *>(data - off) + i * 16);
        return ONCE ? __builtin_nontemporal_load(p) : *p;
    }
    // Any piece, `fill` outside the row.
    template <bool ONCE> __device__ __forceinline__ v4u piece(int i, T fill) const {
        if (i >= first && i < last) return whole<ONCE>(i);
        v4u part{};
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const int index = i * P - off + j;
            const T x = index >= 0 && index < v ? data[index] : fill;
            if constexpr (P == 4)
                part[j] = __builtin_bit_cast(u32, x);
            else
                part[j / 2] |= u32(__builtin_bit_cast(unsigned short, x)) << 16 * (j % 2);
        }
        return part;
    }
};

template <typename T> __device__ __forceinline__ void unpack(v4u raw, float (&x)[PIECE<T>]) {
    // (By shifts: arrays of 16-bit values that live across branches go through memory.)
#pragma unroll
    for (int j = 0; j < PIECE<T>; ++j) {
        if constexpr (PIECE<T> == 4)
            x[j] = __uint_as_float(raw[j]);
        else
            x[j] = float(__builtin_bit_cast(T, static_cast<unsigned short>(raw[j / 2] >> 16 * (j % 2))));
    }
}

template <typename T, int COUNT>
__device__ __forceinline__ void unpack(const v4u (&raw)[COUNT], float (&x)[COUNT][PIECE<T>]) {
#pragma unroll
    for (int t = 0; t < COUNT; ++t) unpack<T>(raw[t], x[t]);
}

// Calls f(i, raw) for this thread's pieces from `start` on: pieces i, i + THREADS, ... four at a
// time, so that as many loads are in flight (with one, a compute unit's waves keep too few bytes under
// way to fill the memory's latency), then singly. Pieces that are not whole come last.
template <int THREADS, bool ONCE, typename T, typename F>
__device__ __forceinline__ void for_pieces(const Row<T> &row, int start, float fill, F f) {
    constexpr int LOADS = 4;
    int i = max(start, row.first) + int(threadIdx.x);
    for (; i + (LOADS - 1) * THREADS < row.last; i += LOADS * THREADS) {
        v4u raw[LOADS];
#pragma unroll
        for (int t = 0; t < LOADS; ++t) raw[t] = row.template whole<ONCE>(i + t * THREADS);
        f(i, raw);
    }
    v4u raw[1];
    for (; i < row.last; i += THREADS) {
        raw[0] = row.template whole<ONCE>(i);
        f(i, raw);
    }
    const int side = threadIdx.x == 0 ? 0 : row.pieces - 1;
    if (threadIdx.x < 2 && side >= start && (side < row.first || side >= row.last) &&
        (threadIdx.x == 0 || row.pieces > 1)) {
        raw[0] = row.template piece<ONCE>(side, T(fill));
        f(side, raw);
    }
}

// The largest of a piece. (v_max3 as it is: fmaxf would first quiet every operand.)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
    return d;
}

template <int P> __device__ __forceinline__ float largest(const float (&x)[P], float top) {
#pragma unroll
    for (int j = 0; j < P; j += 2) top = max3(top, x[j], x[j + 1]);
    return top;
}

// One bit for each class, in the order of the row's pieces.
template <typename T>
__device__ __forceinline__ u32 piece_bits(const u32 *bits, int i) {
    constexpr u32 P = PIECE<T>;
    return bits[u32(i) * P / 32] >> (u32(i) * P % 32) & ((1u << P) - 1u);
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
    const float *norm;       // with a gradient: what the rows' weights are multiplied by
    float inverse_n;         // the same where norm is nullptr
    void *grad;              // [n, v]
    i64 first;               // row of the launch's first workgroup
};

// p d - p + q with d = log(p / q), as p (d + exp(-d) - 1) where that stays in range.
__device__ __forceinline__ double bucket_loss(double p, double q, double d) {
    if (p == 0.0) return q;
    return d > -8.0 ? p * (d + expm1(-d)) : p * d + (q - p);
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

// Writes a piece of the gradient; entries are left to the threads that hold them. `vec`: grad's pieces
// lie at 16-byte addresses as the row's do. (Else, as with a part of a wider matrix's columns, single stores.)
template <typename T>
__device__ __forceinline__ void store_rest(T *grad, const Row<T> &row, int i, u32 marked, bool vec,
                                           const float (&x)[PIECE<T>]) {
    Piece<T> piece;
#pragma unroll
    for (int j = 0; j < PIECE<T>; ++j) piece.v[j] = T(x[j]);
    if (marked == 0 && vec && i >= row.first && i < row.last) {
        // Past the cache, where the logits of rows under way stay (310 -> 272 us for 2048 x 128000 BF16).
        __builtin_nontemporal_store(
            __builtin_bit_cast(v4u, piece),
            reinterpret_cast<v4u *>(reinterpret_cast<char *>(grad - row.off) + i * 16));
    } else {
        const int first = i * PIECE<T> - row.off;
#pragma unroll
        for (int j = 0; j < PIECE<T>; ++j)
            if (first + j >= 0 && first + j < row.v && !(marked >> j & 1u)) grad[first + j] = piece.v[j];
    }
}

// The gradient of a row's classes outside its entries.
template <typename T, int THREADS>
__device__ __forceinline__ void write_rest(const Row<T> &row, const u32 *bits, float c, float ref,
                                           float coef, T *grad) {
    const bool vec = (reinterpret_cast<uintptr_t>(grad - row.off) & 15) == 0;
    if (coef == 0.0f) {   // nothing flows back, whatever the logits are
        const float zero[PIECE<T>] = {};
        for (int i = threadIdx.x; i < row.pieces; i += THREADS)
            store_rest(grad, row, i, piece_bits<T>(bits, i), vec, zero);
        return;
    }
    for_pieces<THREADS, true>(row, 0, 0.0f, [&](int i, auto &raw) {
        constexpr int COUNT = sizeof(raw) / sizeof(raw[0]);
        float x[COUNT][PIECE<T>];
        unpack<T>(raw, x);
#pragma unroll
        for (int t = 0; t < COUNT; ++t) {
#pragma unroll
            for (int j = 0; j < PIECE<T>; ++j) x[t][j] = power(x[t][j], ref, c) * coef;
            store_rest(grad, row, i + t * THREADS, piece_bits<T>(bits, i + t * THREADS), vec, x[t]);
        }
    });
}

// One workgroup a row: one pass over the row for the classes outside the entries, and with GRAD
// another that writes the gradient for an incoming 1. 2048 x 128000 BF16: 110 us for the loss alone
// (4.8 TB/s), 250 with the gradient, for which a copy's rate would take 212. The second pass finds the
// row in the memory's cache, not in an XCD's L2, where the rows under way (16 MB to 4 MB of it) have no
// room: 1.57 GB pass the L2, 6.3 TB/s, and the vector units are busy most of the time. (Rows kept in LDS
// and registers between the passes leave a workgroup a compute unit, and were slower.)
template <typename T, int WAVES, bool GRAD>
__global__ __launch_bounds__(64 * WAVES, 5) void k_distill(const DistillArgs a) {
    extern __shared__ u32 bits[];
    __shared__ __align__(16) float scratch[2 * WAVES];     // two floats or one double a wave
    constexpr int THREADS = 64 * WAVES;
    const i64 r = a.first + blockIdx.x;
    const float weight = a.weight ? a.weight[r] : 1.0f;
    if (weight == 0.0f) {   // nothing of such a row is read
        for (i64 j = threadIdx.x; j < a.k; j += THREADS) a.entry_grad[r * a.k + j] = 0.0f;
        if (threadIdx.x == 0) a.row_loss[r] = a.ref[r] = a.coef[r] = 0.0f;
        if (GRAD)
            for (i64 i = threadIdx.x; i < a.v; i += THREADS) static_cast<T *>(a.grad)[r * a.v + i] = T(0.0f);
        return;
    }
    const T *s = static_cast<const T *>(a.logits) + r * a.ld;
    const i64 first = r * a.k;
    const i64 *indices = a.indices + r * a.k;
    const Row<T> row(s, a.v);
    const float c = LOG2E / a.temperature;
    const bool bad = mark_entries(indices, a.k, a.v, row.off, bits, (row.off + a.v + 31) / 32,
                                  THREADS);

    LogSum rest;
    for_pieces<THREADS, !GRAD>(row, 0, -INFINITY, [&](int i, auto &raw) {
        constexpr int COUNT = sizeof(raw) / sizeof(raw[0]);
        float x[COUNT][PIECE<T>];
        unpack<T>(raw, x);
        float top = rest.m;
#pragma unroll
        for (int t = 0; t < COUNT; ++t) {
            if (const u32 marked = piece_bits<T>(bits, i + t * THREADS)) {
#pragma unroll
                for (int j = 0; j < PIECE<T>; ++j)
                    if (marked >> j & 1u) x[t][j] = -INFINITY;
            }
            top = largest(x[t], top);
        }
        if (top > rest.m) {
            rest.s *= power(rest.m, top, c);
            rest.m = top;
        }
        const float ref = rest.ref();
#pragma unroll
        for (int t = 0; t < COUNT; ++t)
#pragma unroll
            for (int j = 0; j < PIECE<T>; ++j) rest.s += power(x[t][j], ref, c);
    });
    rest = block_merge<WAVES>(rest, c, scratch);

    // The entries and the buckets, k + 1 values a row, are taken in 64 bits: near its teacher, a
    // student's gradient is a small difference of q and p.
    const double cold = 1.0 / double(a.temperature);
    const float tail = a.tail ? a.tail[r] * a.temperature : -INFINITY;   // as a logit
    float most_t = tail, most_z = rest.m;
    for (i64 j = threadIdx.x; j < a.k; j += THREADS)
        if (!bad && indices[j] >= 0) {
            most_t = fmaxf(most_t, value_at(a.values, a.values_type, first + j));
            most_z = fmaxf(most_z, float(s[indices[j]]));
        }
    most_t = block_max<WAVES>(most_t, scratch);
    most_z = block_max<WAVES>(most_z, scratch);
    // What exponents are taken from; -inf stands for values that are all -inf.
    const double t0 = most_t == -INFINITY ? 0.0 : double(most_t);
    const double z0 = most_z == -INFINITY ? 0.0 : double(most_z);
    double teacher = 0.0, student = 0.0;
    for (i64 j = threadIdx.x; j < a.k; j += THREADS)
        if (!bad && indices[j] >= 0) {
            teacher += exp((double(value_at(a.values, a.values_type, first + j)) - t0) * cold);
            student += exp((double(float(s[indices[j]])) - z0) * cold);
        }
    teacher = block_sum<WAVES>(teacher, scratch);
    student = block_sum<WAVES>(student, scratch);
    const double tail_mass = exp((double(tail) - t0) * cold);
    // 0 where nothing is left outside the entries: ref() is then no logit's value, and may be so far above
    // z0 that the exponential is infinite.
    const double rest_scale = rest.s == 0.0f ? 0.0 : exp((double(rest.ref()) - z0) * cold);
    teacher += tail_mass;
    student += rest_scale * double(rest.s);
    const bool empty = most_t == -INFINITY && teacher == 0.0;
    // log(p / q) = ((t - t0) - (z - z0)) / T - shift.
    const double shift = log(teacher) - log(student);
    double loss = 0.0;
    for (i64 j = threadIdx.x; j < a.k; j += THREADS) {
        float grad = 0.0f;
        if (bad) {
            grad = NAN;
        } else if (indices[j] >= 0 && !empty) {
            const double t = (double(value_at(a.values, a.values_type, first + j)) - t0) * cold;
            const double z = (double(float(s[indices[j]])) - z0) * cold;
            const double p = exp(t) / teacher, q = exp(z) / student;
            loss += bucket_loss(p, q, t - z - shift);
            grad = float(q - p);
        }
        a.entry_grad[r * a.k + j] = grad;
    }
    loss = block_sum<WAVES>(loss, scratch);
    float coef = 0.0f;
    if (bad) {                  // and the bucket of all other classes, by every thread
        loss = coef = NAN;
    } else if (!empty) {
        const double p = tail_mass / teacher, scale = rest_scale / student, sum = double(rest.s);
        const double z = (double(rest.ref()) - z0) * cold + log(sum);
        loss += bucket_loss(p, sum * scale, (double(tail) - t0) * cold - z - shift);
        // Without any finite class outside the entries there is nothing to scale.
        coef = sum == 0.0 ? (p > 0.0 ? NAN : 0.0f) : float(scale - p / sum);
    }
    if (threadIdx.x == 0) {
        a.row_loss[r] = float(loss * a.temperature * a.temperature);
        a.ref[r] = rest.ref();
        a.coef[r] = coef;
    }
    if (GRAD) {
        const float scale = 1.0f * weight * (a.norm ? *a.norm : a.inverse_n) * a.temperature;
        T *grad = static_cast<T *>(a.grad) + r * a.v;
        write_rest<T, THREADS>(row, bits, c, rest.ref(), coef * scale, grad);
        for (i64 j = threadIdx.x; j < a.k; j += THREADS) {   // this thread's own entry_grad
            const i64 index = indices[j];
            if (index >= 0 && index < a.v)
                grad[index] = T(bad ? NAN : scale == 0.0f ? 0.0f : a.entry_grad[r * a.k + j] * scale);
        }
    }
}

// sum(weight * loss) over the rows, divided by sum(weight) where `mean`, in a fixed order, in FP64;
// norm = 1 / sum(weight) (0 where there is no weight) or 1. Without row_loss the norm alone.
__global__ __launch_bounds__(256) void k_distill_total(const float *row_loss, const float *weight, i64 n,
                                                       bool mean, float *loss, float *norm) {
    __shared__ double part[2][256];
    double sum = 0.0, weights = 0.0;
    for (i64 r = threadIdx.x; r < n; r += 256) {
        const float w = weight ? weight[r] : 1.0f;
        if (row_loss) sum += double(w) * double(row_loss[r]);
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
        if (row_loss) *loss = total == 0.0 && mean ? 0.0f : float(part[0][0] * scale);
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
    bool unless_one;          // the gradient for an incoming 1 is there already
    void *grad;               // [n, v]
    i64 first;                // row of the launch's first workgroup
};

// The gradient for another incoming value, from the row's reference and coefficient: one pass, bound by
// its bytes (2048 x 128000 BF16 213 us, 1.05 GB at 4.9 TB/s). After a sum or mean it writes what k_distill
// wrote for 1 a second time: forward and backward of a loss times 0.5 465 us, against 260 of the loss itself.
template <typename T, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_distill_grad(const DistillGradArgs a) {
    extern __shared__ u32 bits[];
    constexpr int THREADS = 64 * WAVES;
    const i64 r = a.first + blockIdx.x;
    if (a.unless_one && *a.incoming == 1.0f) return;
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
    write_rest<T, THREADS>(row, bits, c, ref, coef, grad);
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

__device__ __forceinline__ u64 key_of(float x, int index) {
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
    i64 first;            // row of the launch's first workgroup
};

constexpr int TOP_LIST = 2048;      // candidates of a row

struct TopShared {
    u64 list[TOP_LIST];     // in whole steps of rank_list
    u32 ranks[TOP_LIST];
    u64 bounds[16];
    u32 counts[256];
    u32 digit, remaining, found, last;
    alignas(16) float scratch[32];
};

// The value of a key's logit, in FP32; NaN for the largest key.
__device__ __forceinline__ float value_of(u64 key) {
    const u32 order = u32(key >> 32);
    return __uint_as_float(order >> 31 ? order ^ 0x80000000u : ~order);
}

// A thread's listed key is held back until it has another: most have none or one, and those go into the
// list together, with one atomic a wave, instead of one wait for the LDS each.
__device__ __forceinline__ void list_key(TopShared &sh, u64 key) {
    const u32 at = atomicAdd(&sh.found, 1u);
    if (at < u32(TOP_LIST)) sh.list[at] = key;
}

__device__ __forceinline__ void list_pending(TopShared &sh, u64 &pending) {
    const u64 mask = __ballot(pending != 0);
    if (mask == 0) return;
    u32 first = 0;
    if ((threadIdx.x & 63) == 0) first = atomicAdd(&sh.found, u32(__popcll(mask)));
    first = __builtin_amdgcn_readfirstlane(first);
    const u32 at = first + __builtin_amdgcn_mbcnt_hi(u32(mask >> 32), __builtin_amdgcn_mbcnt_lo(u32(mask), 0));
    if (pending != 0 && at < u32(TOP_LIST)) sh.list[at] = pending;
    pending = 0;
}

// What a thread has found in its pieces. A piece with a class from `least` on, the value of the key
// `bound`, is held back whole and looked into when the thread meets another or at the end: most of a
// wave's pieces have such a class in some lane, and going through the classes of each of them took twice
// the instructions of all the rest.
template <typename T> struct Sift {
    static constexpr int P = PIECE<T>;
    float c, b;
    float least;
    u64 bound;
    float sum = 0.0f;       // of exp2(x c + b) over what is not listed
    v4u held{};
    int at = -1;            // which piece is held
    u64 pending = 0;        // a key that is not yet in the list

    // Pieces i, i + step, ... before `end`; those of a row's edges, which the caller knows, are held.
    // A NaN in a piece that is not held makes the sum one.
    template <int COUNT>
    __device__ __forceinline__ void add(const Row<T> &row, TopShared &sh, v4u (&raw)[COUNT], int i,
                                        int step, int end) {
        u32 hold = 0;
#pragma unroll
        for (int t = 0; t < COUNT; ++t) {
            float x[P], part = 0.0f;
            // (Unpacked one after the other: all of them at once take twice the registers.)
            asm volatile("" : "+v"(raw[t]));
            unpack<T>(raw[t], x);
#pragma unroll
            for (int j = 0; j < P; ++j) part += __builtin_amdgcn_exp2f(fmaf(x[j], c, b));
            const int piece = i + t * step;
            if (piece < end) {
                const bool in = largest(x, -INFINITY) >= least || piece < row.first || piece >= row.last;
                hold |= in ? 1u << t : 0u;
                sum += in ? 0.0f : part;
            }
        }
        for (; hold; hold &= hold - 1) {
            if (at >= 0) look(row, sh);
            const int t = __ffs(hold) - 1;
            held = raw[0];
#pragma unroll
            for (int o = 1; o < COUNT; ++o) held = t == o ? raw[o] : held;
            at = i + t * step;
        }
    }
    // Lists the classes of the held piece from `bound` on and adds the others. A NaN is listed.
    __device__ __forceinline__ void look(const Row<T> &row, TopShared &sh) {
        float x[P];
        unpack<T>(held, x);
#pragma unroll
        for (int j = 0; j < P; ++j) {
            bool listed = false;
            if (!(x[j] < least)) {
                const int index = at * P - row.off + j;
                const u64 key = key_of(x[j], index);
                if (index >= 0 && index < row.v && key >= bound) {
                    if (pending != 0) list_key(sh, pending);
                    pending = key;
                    listed = true;
                }
            }
            if (!listed) sum += __builtin_amdgcn_exp2f(fmaf(x[j], c, b));
        }
        at = -1;
    }
    __device__ __forceinline__ void finish(const Row<T> &row, TopShared &sh) {
        if (at >= 0) look(row, sh);
        list_pending(sh, pending);
    }
};

// The smallest selected key by radix selection, eight bits a pass over the row: for rows with
// more than TOP_LIST candidates.
template <typename T, int THREADS>
__device__ u64 exact_bound(const Row<T> row, int k, TopShared &sh) {
    u64 prefix = 0;
    __syncthreads();
    if (threadIdx.x == 0) sh.remaining = k;
    for (int shift = 56;; shift -= 8) {
        __syncthreads();
        for (int b = threadIdx.x; b < 256; b += THREADS) sh.counts[b] = 0;
        __syncthreads();
        for_pieces<THREADS, false>(row, 0, 0.0f, [&](int i, auto &raw) {
#pragma unroll
            for (int t = 0; t < int(sizeof(raw) / sizeof(raw[0])); ++t) {
                float x[PIECE<T>];
                unpack<T>(raw[t], x);
#pragma unroll
                for (int j = 0; j < PIECE<T>; ++j) {
                    const int index = (i + t * THREADS) * PIECE<T> - row.off + j;
                    const u64 key = key_of(x[j], index);
                    if (index >= 0 && index < row.v &&
                        (shift == 56 || key >> (shift + 8) == prefix >> (shift + 8)))
                        atomicAdd(&sh.counts[key >> shift & 255u], 1u);
                }
            }
        });
        __syncthreads();
        if (threadIdx.x == 0) {   // the digit that holds the k-th largest
            u32 left = sh.remaining;
            int d = 255;
            while (sh.counts[d] < left) left -= sh.counts[d--];
            sh.digit = d;
            sh.remaining = left;
            sh.last = sh.counts[d] == left;
        }
        __syncthreads();
        prefix |= u64(sh.digit) << shift;
        if (sh.last || shift == 0) return prefix;
    }
}

// Every listed key's rank among the list, its comparisons shared by several threads, eight at a time.
template <int THREADS> __device__ void rank_list(TopShared &sh, int found) {
    constexpr int STEP = 8;
    const int steps = (found + STEP - 1) / STEP;
    for (int j = threadIdx.x; j < found; j += THREADS) sh.ranks[j] = 0;
    for (int j = found + threadIdx.x; j < steps * STEP; j += THREADS) sh.list[j] = 0;   // above nothing
    __syncthreads();
    const int parts = max(1, min(THREADS / found, steps));
    const int length = (steps + parts - 1) / parts;
    for (int e = threadIdx.x; e < found * parts; e += THREADS) {
        const int j = e % found, from = e / found * length, to = min(from + length, steps);
        const u64 key = sh.list[j];
        u32 above = 0;
        for (int o = from; o < to; ++o)
#pragma unroll
            for (int i = 0; i < STEP; ++i) above += sh.list[o * STEP + i] > key;
        if (parts == 1)
            sh.ranks[j] = above;
        else
            atomicAdd(&sh.ranks[j], above);
    }
    __syncthreads();
}

// The q-th largest key of the wave's lanes, bit by bit; 0 where fewer lanes have one. Keys differ but
// for zeros, and the bits of an index above the 20th are ones.
__device__ __forceinline__ u64 nth_of_wave(u64 key, int q) {
    u64 mask = ~u64(0), prefix = 0;
    int left = q;
    for (int bit = 63; bit >= 0; --bit) {
        const u64 ones = __ballot(key >> bit & 1) & mask;
        const int count = __popcll(ones);
        if (count >= left) {
            mask = ones;
            prefix |= u64(1) << bit;
        } else {
            left -= count;
            mask &= ~ones;
        }
        if (__popcll(mask) == 1) return __shfl((unsigned long long)key, __ffsll((unsigned long long)mask) - 1);
    }
    return prefix;
}

// Sorts the list and leaves its first k keys; the others join the sum, in their order, because the
// order in which they were listed changes from run to run.
template <int THREADS>
__device__ void keep_first(TopShared &sh, int k, float c, float b, float &sum) {
    constexpr int EACH = TOP_LIST / THREADS;
    const int found = int(sh.found);
    rank_list<THREADS>(sh, found);
    u64 keys[EACH];
    u32 ranks[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int j = threadIdx.x + e * THREADS;
        keys[e] = j < found ? sh.list[j] : 0;
        ranks[e] = j < found ? sh.ranks[j] : 0;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < EACH; ++e)
        if (int(threadIdx.x) + e * THREADS < found) sh.list[ranks[e]] = keys[e];
    if (threadIdx.x == 0) sh.found = min(found, k);
    __syncthreads();
    for (int j = k + threadIdx.x; j < found; j += THREADS)
        sum += __builtin_amdgcn_exp2f(fmaf(value_of(sh.list[j]), c, b));
    __syncthreads();
}

// One workgroup a row, as a rule one pass over it. Its first stretch (ITEMS pieces a thread, in registers)
// gives a bound: of the largest classes of a wave's lanes the ceil(k / waves)-th largest, the smallest over
// the waves; at least k classes lie at or above it. Those are listed, and the k-th of the list is the bound
// for the rest of the row, of which it lists about k / (stretch) a class. A listed class's rank is its
// place in the output. Keys hold the index, so ties do not lengthen the list; a row that rises all along
// does, and takes exact_bound's passes over the cached row. So do ordinary rows of large k: the bound comes
// from one class a lane, and where k nears the lanes it is their least, above which lie more classes than
// the list holds. 2048 x 128000 BF16 (us): k = 128 170, 250 248, 512 462, 700 750, and from about 820 on,
// with the exact passes, 1950 to 2180.
// All classes that are not selected are summed relative to the first bound; where that overflows
// or underflows, or the row holds a NaN, once more relative to their own maximum.
// What it costs beyond the bytes (106 us at a copy's rate for 2048 x 128000 BF16, measured 132: 4.0 TB/s;
// a few more under the profiler) are the exponentials, a quarter of the vector units' rate, and the phases in
// which a workgroup ranks and loads nothing, which the others on its compute unit fill.
template <typename T, int WAVES, int ITEMS>
__global__ __launch_bounds__(64 * WAVES, 4) void k_top(const TopArgs a) {
    __shared__ TopShared sh;
    constexpr int THREADS = 64 * WAVES, P = PIECE<T>;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const i64 r = a.first + blockIdx.x;
    const Row<T> row(static_cast<const T *>(a.logits) + r * a.ld, a.v);
    const float c = LOG2E / a.temperature;
    if (threadIdx.x == 0) sh.found = 0;

    // Kept packed: the empty asm keeps the compiler from holding the values unpacked as well, which
    // takes twice the registers.
    v4u first[ITEMS];
    auto values = [&](int t, float (&x)[P]) {
        asm volatile("" : "+v"(first[t]));
        unpack<T>(first[t], x);
    };
#pragma unroll
    for (int t = 0; t < ITEMS; ++t) {
        const int i = threadIdx.x + t * THREADS;
        if (i < row.pieces) first[t] = row.template piece<true>(i, T(-INFINITY));
    }
    // The largest key of this thread (the first of equal ones), 0 for none: its piece, then its place there.
    float top = -INFINITY;
    v4u holder = first[0];
    int at = 0;
#pragma unroll
    for (int t = 0; t < ITEMS; ++t)
        if (int(threadIdx.x) + t * THREADS < row.pieces) {
            float x[P];
            values(t, x);
            const float m = largest(x, -INFINITY);
            if (m > top) {
                top = m;
                holder = first[t];
                at = t;
            }
        }
    u64 best = 0;
    {
        float x[P];
        unpack<T>(holder, x);
        int where = -1;
#pragma unroll
        for (int j = P - 1; j >= 0; --j) where = x[j] == top ? j : where;
        const int i = threadIdx.x + at * THREADS, index = i * P - row.off + where;
        if (i < row.pieces && where >= 0 && index >= 0 && index < row.v) best = key_of(top, index);
    }
    const int full = min(WAVES, row.pieces / 64);       // waves with a piece in every lane
    const bool bounded = a.k <= 64 * full;
    if (bounded && wave < full) {
        const u64 mine = nth_of_wave(best, (a.k + full - 1) / full);
        if (lane == 0) sh.bounds[wave] = mine;
    }
    __syncthreads();
    u64 bound = bounded ? sh.bounds[0] : 0;
#pragma unroll
    for (int w = 1; w < WAVES; ++w)
        if (bounded && w < full) bound = min(bound, sh.bounds[w]);

    const float least = bound ? value_of(bound) : -INFINITY;      // 0 lists everything
    const float b = least == -INFINITY ? 0.0f : -least * c;
    Sift<T> sift{c, b, least, bound};
    // All pieces together where rows fill the chip (133 against 152 us for 2048 x 128000 BF16), four at a
    // time for few rows (15.0 against 16.4 us for 1 x 50001 FP32).
    constexpr int LOADS = 4, TOGETHER = WAVES < 16 ? ITEMS : LOADS;
#pragma unroll
    for (int t = 0; t < ITEMS; t += TOGETHER)
        sift.add(row, sh, reinterpret_cast<v4u (&)[TOGETHER]>(first[t]), threadIdx.x + t * THREADS,
                 THREADS, row.pieces);
    sift.finish(row, sh);
    // A NaN is found by the sum: it may be among the largest, which comparisons of values miss.
    bool exact = __syncthreads_or(sift.sum != sift.sum) || sh.found > u32(TOP_LIST);
    if (!exact && row.pieces > ITEMS * THREADS) {
        keep_first<THREADS>(sh, a.k, c, b, sift.sum);
        sift.bound = sh.list[a.k - 1];
        sift.least = value_of(sift.bound);
        if (threadIdx.x == 0 && row.last < row.pieces) {
            sift.held = row.template piece<true>(row.last, T(-INFINITY));
            sift.at = row.last;
        }
        for (int i = ITEMS * THREADS + threadIdx.x; i < row.last; i += LOADS * THREADS) {
            v4u raw[LOADS]{};
#pragma unroll
            for (int t = 0; t < LOADS; ++t)
                if (i + t * THREADS < row.last) raw[t] = row.template whole<true>(i + t * THREADS);
            sift.add(row, sh, raw, i, THREADS, row.last);
        }
        sift.finish(row, sh);
        exact = __syncthreads_or(sift.sum != sift.sum) || sh.found > u32(TOP_LIST);
    }
    if (exact) {
        const Row<T> again = row;
        bound = exact_bound<T, THREADS>(again, a.k, sh);      // lists k classes
        if (threadIdx.x == 0) sh.found = 0;
        __syncthreads();
        float others = 0.0f;
        for_pieces<THREADS, false>(again, 0, -INFINITY, [&](int i, auto &raw) {
#pragma unroll
            for (int t = 0; t < int(sizeof(raw) / sizeof(raw[0])); ++t) {
                float x[P];
                unpack<T>(raw[t], x);
#pragma unroll
                for (int j = 0; j < P; ++j) {
                    const int index = (i + t * THREADS) * P - again.off + j;
                    const u64 key = key_of(x[j], index);
                    if (index >= 0 && index < again.v && key >= bound)
                        list_key(sh, key);
                    else
                        others += __builtin_amdgcn_exp2f(fmaf(x[j], c, b));
                }
            }
        });
        sift.sum = others;
        __syncthreads();
    }
    float sum = sift.sum;
    keep_first<THREADS>(sh, a.k, c, b, sum);
    for (int j = threadIdx.x; j < a.k; j += THREADS) {
        const int index = int(0xffffffffu - u32(sh.list[j]));
        a.indices[r * a.k + j] = index;
        static_cast<T *>(a.values)[r * a.k + j] = row.data[index];
    }

    sum = block_sum<WAVES>(sum, sh.scratch);
    float tail = (__builtin_amdgcn_logf(sum) - b) * LN2;
    if (a.k < a.v && !(sum > 0x1p-60f && sum < 0x1p60f && fabsf(b) < 0x1p60f)) {
        const u64 last = sh.list[a.k - 1];
        const Row<T> again = row;
        LogSum rest;
        bool infinite = false, nan = false;
        for_pieces<THREADS, false>(again, 0, -INFINITY, [&](int i, auto &raw) {
#pragma unroll
            for (int t = 0; t < int(sizeof(raw) / sizeof(raw[0])); ++t) {
                float x[P];
                unpack<T>(raw[t], x);
#pragma unroll
                for (int j = 0; j < P; ++j) {
                    const int index = (i + t * THREADS) * P - again.off + j;
                    if (index < 0 || index >= again.v || key_of(x[j], index) >= last) continue;
                    infinite = infinite || x[j] == INFINITY;
                    nan = nan || x[j] != x[j];
                    rest.add(x[j], c);
                }
            }
        });
        rest = block_merge<WAVES>(rest, c, sh.scratch);
        // A +inf makes the tail +inf, where the sum relative to it is NaN; a NaN makes it NaN.
        infinite = __syncthreads_or(infinite);
        nan = __syncthreads_or(nan);
        if (infinite && !nan)
            tail = INFINITY;
        else if (rest.m == -INFINITY && rest.s == 0.0f)
            tail = -INFINITY;
        else
            tail = rest.ref() / a.temperature + __builtin_amdgcn_logf(rest.s) * LN2;
    }
    if (threadIdx.x == 0) a.tail[r] = a.k < a.v ? tail : -INFINITY;
}

// (log2(e) / T is finite from FLT_MIN on.)
static int check_rows(const char *what, const void *logits, int32_t type, i64 n, i64 v, i64 ld, i64 k,
                      float temperature) {
    if (!logits || !known_type(type) || n < 1 || v < 1 || k < 1 || k > v || (n > 1 && ld < v) ||
        !(temperature >= FLT_MIN) || !(temperature <= FLT_MAX) || !aligned(logits, type_bytes(type)))
        return fail(MF_E_INVALID, "invalid %s arguments", what);
    if (v > MOST_CLASSES || n > i64(1) << 30)
        return fail(MF_E_UNSUPPORTED, "%s takes at most %lld classes and %lld rows", what,
                    (long long)MOST_CLASSES, (long long)(i64(1) << 30));
    if (k > MOST_ENTRIES)
        return fail(MF_E_UNSUPPORTED, "%s takes at most %d entries a row", what, MOST_ENTRIES);
    return MF_OK;
}

constexpr int ROW_WAVES = 8;

// Launches a workgroup a row. A launch has fewer than 2^32 threads, so more rows take several.
template <typename K, typename A>
static int launch_rows(const char *what, K kernel, A args, int waves, size_t lds, hipStream_t s) {
    constexpr i64 ROWS = i64(1) << 21;      // of at most 1024 threads
    for (args.first = 0; args.first < args.n; args.first += ROWS) {
        hipLaunchKernelGGL(kernel, dim3(unsigned(std::min(ROWS, args.n - args.first))), dim3(64 * waves), lds,
                           s, args);
        if (const int status = check_launch(what)) return status;
    }
    return MF_OK;
}

static size_t mark_bytes(i64 v) { return size_t((v + 8 + 31) / 32 * 4); }

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
        // Few rows take sixteen waves each (us, 64 x 128000 BF16, k = 64, 4 / 8 / 16 waves: 49 / 30 / 27), of
        // which a compute unit holds one workgroup: 256 rows 30, 300 rows 49, 511 rows 56 and 512 57.
        // Where the rows fill the chip, small workgroups let some list while others load; a longer
        // stretch and more waves pay where the bound would list many classes, and a wave's bound is near
        // the row's while k is at most half its lanes times the waves (us, 2048 rows BF16, four waves of 8
        // and of 16 pieces / eight of 16: 16000 classes, k = 64 41 / 44 / 68; 128000, k = 64 206 / 132 / 141;
        // 128000, k = 128 380 / 195 / 174; between them k * v is drawn from these alone).
        const i64 pieces = v / PIECE<T>;
        const auto launch = [&](auto kernel, int waves) {
            return launch_rows("top logits", kernel, args, waves, 0, static_cast<hipStream_t>(stream));
        };
        if (n < 512 ? pieces >= 1024 || k > 128 : k > 256) return launch(k_top<T, 16, 16>, 16);
        if (k <= 128 && pieces <= 4 * 64 * 8) return launch(k_top<T, 4, 8>, 4);
        if (k <= 128 && k * v <= 256 * 4096 * PIECE<T>) return launch(k_top<T, 4, 16>, 4);
        return launch(k_top<T, 8, 16>, 8);
    });
}

int mf_distill_loss(const void *logits, int32_t type, int64_t n, int64_t v, int64_t ld,
                    const void *values, int32_t values_type, const int64_t *indices,
                    const float *tail, int64_t k, float temperature, const float *weight,
                    int32_t reduction, float *row_loss, float *ref, float *coef, float *entry_grad,
                    float *loss, float *norm, void *grad, void *stream) {
    const int status = check_rows("distillation", logits, type, n, v, ld, k, temperature);
    if (status) return status;
    if (!values || !known_type(values_type) || !indices || !row_loss || !ref || !coef || !entry_grad ||
        reduction < 0 || reduction > 2 || (reduction != MF_SUM_NONE && (!loss || !norm)) ||
        (reduction == MF_SUM_NONE && grad))
        return fail(MF_E_INVALID, "invalid distillation arguments");
    hipStream_t s = static_cast<hipStream_t>(stream);
    DistillArgs args{logits, values, values_type, indices, tail, weight, n, v, ld, k,
                     temperature, row_loss, ref, coef, entry_grad};
    const bool mean = reduction == MF_SUM_MEAN;
    args.grad = grad;
    args.inverse_n = mean ? float(1.0 / double(n)) : 1.0f;
    if (grad && weight && mean) {
        args.norm = norm;
        hipLaunchKernelGGL(k_distill_total, dim3(1), dim3(256), 0, s, nullptr, weight, n, true,
                           nullptr, norm);
    }
    const int launched = with_type(type, [&](auto zero) {
        using T = decltype(zero);
        auto kernel = grad ? k_distill<T, ROW_WAVES, true> : k_distill<T, ROW_WAVES, false>;
        const int lds = allow_lds(kernel, mark_bytes(v));
        if (lds) return lds;
        return launch_rows("distillation loss", kernel, args, ROW_WAVES, mark_bytes(v), s);
    });
    if (launched || reduction == MF_SUM_NONE) return launched;
    hipLaunchKernelGGL(k_distill_total, dim3(1), dim3(256), 0, s, row_loss, weight, n, mean, loss, norm);
    return check_launch("distillation total");
}

int mf_distill_grad(const void *logits, int32_t type, int64_t n, int64_t v, int64_t ld,
                    const int64_t *indices, int64_t k, float temperature, const float *weight,
                    const float *ref, const float *coef, const float *entry_grad, const float *norm,
                    const float *incoming, int64_t incoming_step, int32_t unless_one, void *grad,
                    void *stream) {
    const int status = check_rows("distillation gradient", logits, type, n, v, ld, k, temperature);
    if (status) return status;
    if (!indices || !ref || !coef || !entry_grad || !incoming || !grad || incoming_step < 0 ||
        (unless_one && incoming_step))
        return fail(MF_E_INVALID, "invalid distillation gradient arguments");
    const DistillGradArgs args{logits, indices, weight, ref, coef, entry_grad, norm, incoming,
                               incoming_step, n, v, ld, k, temperature, unless_one != 0, grad};
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        const int lds = allow_lds(k_distill_grad<T, ROW_WAVES>, mark_bytes(v));
        if (lds) return lds;
        return launch_rows("distillation gradient", k_distill_grad<T, ROW_WAVES>, args, ROW_WAVES,
                           mark_bytes(v), static_cast<hipStream_t>(stream));
    });
}

}  // extern "C"
