// Gated linear recurrence over long sequences, and its gradients.
//
//   u = sigmoid(g), k = 1 - u = sigmoid(-g), c = tanh(v) or v,  h_t = u_t h_{t-1} + k_t c_t
// for every channel by itself: a GRU without hidden projections.  A stretch of steps maps the state
// before it to the one after it as h -> A h + S with A the product of its u, and the gradient of
// the state after it to that of the one before it as r -> A r + Q, so stretches are reduced each by
// itself and joined in order:
//   G_t = dy_t + u_{t+1} G_{t+1},  dg_t = G_t (h_{t-1} - c_t) u_t k_t,  dv_t = G_t k_t (1 - c_t^2).
// States, A, S and Q are FP32, whatever the type of g, v and y.
#include <algorithm>
#include <type_traits>

#include "mf_float.h"

namespace mf {

// A wave takes 64 channels and CHUNK steps of them, the up to WAVES waves of a workgroup consecutive chunks,
// whose maps they exchange in LDS. States are kept every SPAN steps for the gradients, which is what a
// workgroup of either shape takes at a time: eight waves of 16 steps, and for sequences that are no longer
// sixteen of 8.
constexpr int SPAN = 128, MOST_WAVES = 16;
constexpr float LOG2E = 1.44269504f, LN2 = 0.693147181f;

struct RecurrenceArgs {
    const void *x;          // [steps, batch, 2 width]: gates, then candidates
    i64 xt, xb;             // distances of steps and of sequences
    const float *state;     // [batch, width] or nullptr: zeros
    const i64 *lengths;     // [batch] or nullptr
    i64 steps, width;
    i64 first, batch, tiles;    // sequences of this launch, and channel tiles of each
    bool reverse;
    void *y;                // out [steps, batch, width], or its gradient (nullptr: zeros)
    i64 yt, yb;
    float *last;            // [batch, width]: the last state, or its gradient (nullptr: zeros)
    float *marks;           // [ceil(steps / SPAN), batch, width]: states before every SPAN steps
    void *dx;               // [steps, batch, 2 width]
    i64 dt, db;
    float *dstate;          // [batch, width] or nullptr
    i64 segments, segment;  // workgroups along the steps, and the steps of each
    float *parts;           // [segments, batch, 2, width]: A and S (or Q) of every segment
    i64 all;                // sequences of the call
};

template <typename T, int V> struct alignas(sizeof(T) * V) Group {
    T v[V];
};

// sigmoid(g) and sigmoid(-g) as u = 1 / (1 + e) and k = e u with e = exp(-g): no difference of near numbers
// at either end. What the rounding of g log2(e) took from the exponent is made good, so that k keeps its
// digits for far gates too, and the reciprocal (within an ulp) is refined to a rounding, since hundreds of u are
// multiplied where a channel remembers long: without it the gradient of the first state is off by up to 1e-6
// after 4096 steps, with it by 2.5e-7 (8 x 4096 x 2048 with gradients 251 -> 256 us). For gates within FAR_GATE,
// where e and u are normal numbers of FP32, which is all that these instructions give; a NaN gives NaN.
constexpr float FAR_GATE = 87.0f, FAR_VALUE = 1.64581143e-38f;     // exp(-87)

__device__ __forceinline__ void gates(float g, float &u, float &k) {
    const float t = g * -LOG2E, rest = fmaf(g, -LOG2E, -t);
    float e = __builtin_amdgcn_exp2f(t);
    e = fmaf(e, rest * LN2, e);
    const float d = 1.0f + e, r = __builtin_amdgcn_rcpf(d);
    u = fmaf(r, fmaf(-d, r, 1.0f), r);
    k = e * u;
}

// Puts in their place what they are for a gate beyond: the smaller exp(-|g|), subnormal numbers and then 0, so that a
// closed gate drops a state of any size, and the other 1. Others are left. A wave comes here where one of its lanes
// has such a gate: 8 x 4096 x 2048 BF16 with one gate in a hundred closed, which is all waves, 123 us for 100.
__device__ __forceinline__ void far_gates(float g, float &u, float &k) {
    const float least = FAR_VALUE * __builtin_amdgcn_exp2f((FAR_GATE - fabsf(g)) * LOG2E);
    const bool far = fabsf(g) > FAR_GATE, closed = g < 0.0f;
    u = far ? (closed ? least : 1.0f) : u;
    k = far ? (closed ? 1.0f : least) : k;
}

// The largest of |g| so far, NaN once there was one; and whether a wave has gates beyond FAR_GATE (or NaN).
__device__ __forceinline__ float farthest(float most, float g) {
    return __builtin_elementwise_maximum(most, fabsf(g));
}
__device__ __forceinline__ bool any_far(float most) { return __builtin_expect(__any(!(most <= FAR_GATE)), 0); }

// Products of u are 0 only where one of their factors is: what gets beneath FP32 is held at its smallest number, so
// that an infinite state stays infinite, as it does step by step, and no finite one is off by more than 2^-149 of
// itself. Of two such products (a NaN is passed on), and of a wave's u, whose plain product is A.
constexpr float SMALLEST = 0x1p-149f;

__device__ __forceinline__ float joined(float a, float b) {
    const float least = __builtin_elementwise_minimum(__builtin_elementwise_minimum(a, b), SMALLEST);
    return __builtin_elementwise_maximum(a * b, least);
}
template <int N> __device__ __forceinline__ float product(float A, const float (&u)[N]) {
    if (__builtin_expect(A == 0.0f, 0)) {
        bool closed = false;
#pragma unroll
        for (int i = 0; i < N; ++i) closed |= u[i] == 0.0f;
        A = closed ? 0.0f : SMALLEST;
    }
    return A;
}

// tanh: 1 - 2 / (1 + exp(2 x)), and where that difference would lose digits the series
// x - x^3 / 3 + 2 x^5 / 15 - 17 x^7 / 315 + 62 x^9 / 2835 (below 1/4 the next term is under 1e-8 of it). The
// reciprocal is not refined: tanh's error does not grow over the steps.
__device__ __forceinline__ float hyperbolic_tangent(float x) {
    const float e = __builtin_amdgcn_exp2f(x * (2.0f * LOG2E));
    const float far = fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + e), 1.0f);
    const float s = x * x;
    float p = fmaf(s, 62.0f / 2835.0f, -17.0f / 315.0f);
    p = fmaf(s, p, 2.0f / 15.0f);
    p = fmaf(s, p, -1.0f / 3.0f);
    return fabsf(x) < 0.25f ? fmaf(x * s, p, x) : far;
}

// What one workgroup works on. All but the channel is the same for a wave, so that addresses are scalar
// but for the lane's own offset in a row, in bytes.
template <typename T, int V> struct Place {
    i64 b, segment, length, begin, end;
    u32 channel, lane_bytes;
    bool inside, reverse;

    __device__ __forceinline__ explicit Place(const RecurrenceArgs &a) : reverse(a.reverse) {
        u32 id = blockIdx.x;
        const u32 tile = id % u32(a.tiles);
        id /= u32(a.tiles);
        b = a.first + id % u32(a.batch);
        segment = id / u32(a.batch);
        const u32 c = (tile * 64 + (threadIdx.x & 63)) * V;
        inside = c < a.width;
        channel = inside ? c : 0;
        lane_bytes = channel * u32(sizeof(T));
        length = a.steps;
        if (a.lengths) {
            length = a.lengths[b];
            length = length < 0 ? 0 : length > a.steps ? a.steps : length;
        }
        begin = segment * a.segment;
        end = min(begin + a.segment, a.steps);
    }
    // Step s of the recurrence lies at time s, or in reverse at length - 1 - s.
    __device__ __forceinline__ i64 time(i64 s) const { return reverse ? length - 1 - s : s; }
    __device__ __forceinline__ i64 at(const RecurrenceArgs &a) const { return b * a.width + channel; }
};

// The rows of one tensor that a workgroup goes through: step s lies `step` bytes behind step s - 1.
template <typename T, int V> struct Rows {
    char *first;        // of step 0
    i64 step;
    __device__ __forceinline__ Rows(const void *p, const Place<T, V> &place, i64 sequence, i64 distance)
        : first(static_cast<char *>(const_cast<void *>(p)) +
                (place.b * sequence + place.time(0) * distance) * i64(sizeof(T))),
          step((place.reverse ? -distance : distance) * i64(sizeof(T))) {}
    __device__ __forceinline__ char *at(i64 s) const { return first + s * step; }
};

template <typename G> __device__ __forceinline__ G get(const char *row, u32 bytes) {
    return *reinterpret_cast<const G *>(row + bytes);
}
template <typename G> __device__ __forceinline__ void put(char *row, u32 bytes, G v) {
    *reinterpret_cast<G *>(row + bytes) = v;
}

// f(i, row) for the CHUNK rows of steps s + i. Rows past the last step are the last one's, which exists
// (length > 0): what they give is left out later.
template <int CHUNK, typename T, int V, typename F>
__device__ __forceinline__ void each_row(const Rows<T, V> &rows, i64 s, i64 length, F f) {
    if (s + CHUNK <= length) {
        char *row = rows.at(s);
#pragma unroll
        for (int i = 0; i < CHUNK; ++i, row += rows.step) f(i, row);
    } else {
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) f(i, rows.at(min(s + i, length - 1)));
    }
}

// The same for the steps that exist alone.
template <int CHUNK, typename T, int V, typename F>
__device__ __forceinline__ void each_step(const Rows<T, V> &rows, i64 s, i64 length, F f) {
    char *row = rows.at(s);
    if (s + CHUNK <= length) {
#pragma unroll
        for (int i = 0; i < CHUNK; ++i, row += rows.step) f(i, row);
    } else {
#pragma unroll
        for (int i = 0; i < CHUNK; ++i, row += rows.step)
            if (s + i < length) f(i, row);
    }
}

__device__ __forceinline__ int wave_of_thread() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// carry through the maps of the segments first .. last - 1, in order (BACK: from the last on): every
// wave composes its share, whose loads it has under way together, and the shares meet in LDS.
template <int V, bool BACK>
__device__ __forceinline__ void fold(const RecurrenceArgs &a, i64 b, i64 channel, i64 first, i64 last,
                                     float (*maps)[2][64 * V], float (&carry)[V]) {
    const int lane = threadIdx.x & 63, wave = wave_of_thread(), waves = blockDim.x >> 6;
    const i64 share = (last - first + waves - 1) / waves;
    const i64 from = min(first + wave * share, last), to = min(from + share, last);
    float A[V], S[V];
#pragma unroll
    for (int j = 0; j < V; ++j) A[j] = 1.0f, S[j] = 0.0f;
    for (i64 n = 0; n < to - from; n += 8) {
        float pa[8][V], ps[8][V];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const i64 z = min(n + i, to - from - 1);
            const float *part = a.parts + (((BACK ? to - 1 - z : from + z) * a.all + b) * 2) * a.width +
                                channel;
#pragma unroll
            for (int j = 0; j < V; ++j) pa[i][j] = part[j], ps[i][j] = part[a.width + j];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const bool live = n + i < to - from;
                A[j] = joined(A[j], live ? pa[i][j] : 1.0f);
                S[j] = live ? fmaf(pa[i][j], S[j], ps[i][j]) : S[j];
            }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        maps[wave][0][lane * V + j] = A[j];
        maps[wave][1][lane * V + j] = S[j];
    }
    __syncthreads();
    for (int n = 0; n < waves; ++n) {
        const int w = BACK ? waves - 1 - n : n;
#pragma unroll
        for (int j = 0; j < V; ++j)
            carry[j] = fmaf(maps[w][0][lane * V + j], carry[j], maps[w][1][lane * V + j]);
    }
    __syncthreads();
}

// Writes zeros at the times from the sequence's length on, in rows `distance` values apart, and where
// `second` is not 0 again that many bytes further.
template <typename T>
__device__ __forceinline__ void blank(const Place<T, 1> &p, void *rows, i64 sequence, i64 distance, int wave,
                                      int waves, u32 second) {
    if (!p.inside) return;
    for (i64 t = max(p.begin, p.length) + wave; t < p.end; t += waves) {
        char *row = static_cast<char *>(rows) + (p.b * sequence + t * distance) * i64(sizeof(T));
        put(row, p.lane_bytes, T(0.0f));
        if (second) put(row, p.lane_bytes + second, T(0.0f));
    }
}

// Bound by its bytes and by the vector units, which are busy two thirds of the time: 8 x 4096 x 2048 BF16 in
// 100 us (403 MB, 4.0 TB/s). Two channels a lane, for wider rows of loads, took 104; sixteen waves of eight
// steps, which join twice as many maps, 115.
template <typename T, bool TANH, int WAVES, int CHUNK>
__global__ __launch_bounds__(64 * WAVES) void k_recurrence(const RecurrenceArgs a) {
    __shared__ float maps[2][WAVES][2][64];
    const Place<T, 1> p(a);
    const int lane = threadIdx.x & 63, wave = wave_of_thread(), waves = blockDim.x >> 6;
    const int span = waves * CHUNK;
    const u32 second = p.lane_bytes + u32(a.width) * u32(sizeof(T));
    const Rows<T, 1> x(a.x, p, a.xb, a.xt), y(a.y, p, a.yb, a.yt);
    const i64 end = min(p.end, p.length);

    T next_g[CHUNK], next_v[CHUNK];
    const auto load = [&](i64 s) {
        each_row<CHUNK>(x, s, p.length, [&](int i, const char *row) {
            next_g[i] = get<T>(row, p.lane_bytes);
            next_v[i] = get<T>(row, second);
        });
    };
    if (p.begin < end) load(p.begin + wave * CHUNK);
    float carry[1] = {a.state ? a.state[p.at(a)] : 0.0f};
    // The state before this segment: the maps of those before it, in order.
    if (p.segment) fold<1, false>(a, p.b, p.channel, 0, p.segment, maps[0], carry);

    int turn = 0;
    for (i64 base = p.begin; base < end; base += span, turn ^= 1) {
        const i64 s = base + wave * CHUNK;
        float u[CHUNK], k[CHUNK], in[CHUNK], A = 1.0f, S = 0.0f, most = 0.0f, h;
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) {
            most = farthest(most, float(next_g[i]));
            gates(float(next_g[i]), u[i], k[i]);
            in[i] = float(next_v[i]);
            if (TANH) in[i] = hyperbolic_tangent(in[i]);
        }
        if (any_far(most))
#pragma unroll
            for (int i = 0; i < CHUNK; ++i) far_gates(float(next_g[i]), u[i], k[i]);
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) in[i] *= k[i];
        if (__builtin_expect(s + CHUNK > p.length, 0))
#pragma unroll
            for (int i = 0; i < CHUNK; ++i)
                if (s + i >= p.length) u[i] = 1.0f, in[i] = 0.0f;
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) {
            A *= u[i];
            S = fmaf(u[i], S, in[i]);
        }
        A = product(A, u);
        if (base + span < end) load(s + span);
        maps[turn][wave][0][lane] = A;
        maps[turn][wave][1][lane] = S;
        __syncthreads();    // one a turn: the other turn's maps are read before its barrier
        for (int w = 0; w < waves; ++w) {
            if (w == wave) h = carry[0];
            carry[0] = fmaf(maps[turn][w][0][lane], carry[0], maps[turn][w][1][lane]);
        }
        if (a.marks && s % SPAN == 0 && s < p.length && p.inside)
            a.marks[s / SPAN * a.all * a.width + p.at(a)] = h;
        T out[CHUNK];
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) {
            h = fmaf(u[i], h, in[i]);
            out[i] = rounded<T>(h);
        }
        if (p.inside)
            each_step<CHUNK>(y, s, p.length, [&](int i, char *row) { put(row, p.lane_bytes, out[i]); });
    }
    blank(p, a.y, a.yb, a.yt, wave, waves, 0);
    if (wave == 0 && p.inside && p.segment == a.segments - 1) a.last[p.at(a)] = carry[0];
}

// As above: 8 x 4096 x 2048 BF16 in 155 us (671 MB, 4.3 TB/s), with sixteen waves of eight steps 175. Two
// channels a lane need more registers than there are.
template <typename T, bool TANH, int WAVES, int CHUNK>
__global__ __launch_bounds__(64 * WAVES) void k_recurrence_grad(const RecurrenceArgs a) {
    __shared__ float maps[2][WAVES][3][64];
    const Place<T, 1> p(a);
    const int lane = threadIdx.x & 63, wave = wave_of_thread(), waves = blockDim.x >> 6;
    const int span = waves * CHUNK;
    const u32 second = p.lane_bytes + u32(a.width) * u32(sizeof(T));
    const Rows<T, 1> x(a.x, p, a.xb, a.xt), dy(a.y, p, a.yb, a.yt), dx(a.dx, p, a.db, a.dt);
    const i64 end = min(p.end, p.length);

    T next_g[CHUNK], next_v[CHUNK], next_dy[CHUNK];
    float mark;
    const auto load = [&](i64 base) {
        const i64 s = base + wave * CHUNK;
        each_row<CHUNK>(x, s, p.length, [&](int i, const char *row) {
            next_g[i] = get<T>(row, p.lane_bytes);
            next_v[i] = get<T>(row, second);
        });
        if (a.y)
            each_row<CHUNK>(dy, s, p.length,
                            [&](int i, const char *row) { next_dy[i] = get<T>(row, p.lane_bytes); });
        mark = a.marks[(base / SPAN * a.all) * a.width + p.at(a)];
    };
#pragma unroll
    for (int i = 0; i < CHUNK; ++i) next_dy[i] = T(0.0f);
    const i64 top = p.begin + (end - p.begin - 1) / span * span;
    if (p.begin < end) load(top);
    // The gradient of the state after this segment: the maps of those behind it, from the last on.
    float carry[1] = {a.last ? a.last[p.at(a)] : 0.0f};
    if (p.segment + 1 < a.segments)
        fold<1, true>(a, p.b, p.channel, p.segment + 1, a.segments,
                      reinterpret_cast<float (*)[2][64]>(&maps), carry);

    int turn = 0;
    if (p.begin < end)
        for (i64 base = top; base >= p.begin; base -= span, turn ^= 1) {
            const i64 s = base + wave * CHUNK;
            float u[CHUNK], k[CHUNK], c[CHUNK], g[CHUNK], A = 1.0f, S = 0.0f, Q = 0.0f, h = mark, r;
            float most = 0.0f;
#pragma unroll
            for (int i = 0; i < CHUNK; ++i) {
                most = farthest(most, float(next_g[i]));
                gates(float(next_g[i]), u[i], k[i]);
                c[i] = float(next_v[i]);
                if (TANH) c[i] = hyperbolic_tangent(c[i]);
                g[i] = float(next_dy[i]);
            }
            if (any_far(most))
#pragma unroll
                for (int i = 0; i < CHUNK; ++i) far_gates(float(next_g[i]), u[i], k[i]);
            if (__builtin_expect(s + CHUNK > p.length, 0))
#pragma unroll
                for (int i = 0; i < CHUNK; ++i)
                    if (s + i >= p.length) u[i] = 1.0f, k[i] = 0.0f, c[i] = 0.0f, g[i] = 0.0f;
#pragma unroll
            for (int i = 0; i < CHUNK; ++i) {
                A *= u[i];
                S = fmaf(u[i], S, k[i] * c[i]);
            }
            A = product(A, u);
#pragma unroll
            for (int i = CHUNK - 1; i >= 0; --i) Q = u[i] * (g[i] + Q);
            if (base > p.begin) load(base - span);
            maps[turn][wave][0][lane] = A;
            maps[turn][wave][1][lane] = S;
            maps[turn][wave][2][lane] = Q;
            __syncthreads();
            for (int w = 0; w < wave; ++w) h = fmaf(maps[turn][w][0][lane], h, maps[turn][w][1][lane]);
            for (int w = waves - 1; w >= 0; --w) {
                if (w == wave) r = carry[0];
                carry[0] = fmaf(maps[turn][w][0][lane], carry[0], maps[turn][w][2][lane]);
            }
            // Factors of G in both gradients, then G from the last step back.
#pragma unroll
            for (int i = 0; i < CHUNK; ++i) {
                const float before = h;
                h = fmaf(u[i], before, k[i] * c[i]);
                const float dv = TANH ? k[i] * fmaf(-c[i], c[i], 1.0f) : k[i];
                c[i] = (before - c[i]) * (u[i] * k[i]);
                k[i] = dv;
            }
            T dg[CHUNK], dv[CHUNK];
#pragma unroll
            for (int i = CHUNK - 1; i >= 0; --i) {
                const float G = g[i] + r;
                dg[i] = rounded<T>(G * c[i]);
                dv[i] = rounded<T>(G * k[i]);
                r = u[i] * G;
            }
            if (p.inside)
                each_step<CHUNK>(dx, s, p.length, [&](int i, char *row) {
                    put(row, p.lane_bytes, dg[i]);
                    put(row, second, dv[i]);
                });
        }
    blank(p, a.dx, a.db, a.dt, wave, waves, u32(a.width) * u32(sizeof(T)));
    if (a.dstate && wave == 0 && p.inside && p.segment == 0) a.dstate[p.at(a)] = carry[0];
}

// A and S of every segment but the last (GRAD: A and Q of every segment but the first), each wave its
// share of the segment's steps. Bound by its bytes and the vector units: 65536 x 512 BF16 in 32 us (134 MB,
// 4.2 TB/s); the segments' own pass reads them again (42 us with the states written).
template <typename T, int V, bool TANH, bool GRAD>
__global__ __launch_bounds__(64 * MOST_WAVES) void k_recurrence_parts(const RecurrenceArgs a) {
    constexpr int CHUNK = 8;
    __shared__ float maps[MOST_WAVES][2][64 * V];
    const Place<T, V> p(a);
    if (p.segment == (GRAD ? 0 : a.segments - 1)) return;
    const int lane = threadIdx.x & 63, wave = wave_of_thread(), waves = blockDim.x >> 6;
    const u32 second = p.lane_bytes + u32(a.width) * u32(sizeof(T));
    const Rows<T, V> x(a.x, p, a.xb, a.xt), dy(a.y, p, a.yb, a.yt);
    const i64 share = a.segment / waves, end = min(p.begin + (wave + 1) * share, p.length);
    float A[V], S[V], low[V];       // low: the least u
#pragma unroll
    for (int j = 0; j < V; ++j) A[j] = low[j] = 1.0f, S[j] = 0.0f;
    for (i64 s = p.begin + wave * share; s < end; s += CHUNK) {
        Group<T, V> g[CHUNK], v[CHUNK];
        each_row<CHUNK>(x, s, p.length, [&](int i, const char *row) {
            g[i] = get<Group<T, V>>(row, p.lane_bytes);
            v[i] = GRAD ? Group<T, V>{} : get<Group<T, V>>(row, second);
        });
        if (GRAD && a.y)
            each_row<CHUNK>(dy, s, p.length,
                            [&](int i, const char *row) { v[i] = get<Group<T, V>>(row, p.lane_bytes); });
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < CHUNK; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) most = farthest(most, float(g[i].v[j]));
        // What a step adds, and the maps of the share with it (GRAD: r -> A u (dy + r) + S).
        const auto added = [&](float k, float c) { return GRAD ? c : k * (TANH ? hyperbolic_tangent(c) : c); };
        const auto step = [&](int j, float u, float add) {
            A[j] = GRAD ? joined(A[j], u) : A[j] * u;
            S[j] = GRAD ? fmaf(A[j], add, S[j]) : fmaf(u, S[j], add);
            low[j] = __builtin_elementwise_minimum(low[j], u);
        };
        const auto steps = [&](auto far) {
#pragma unroll
            for (int i = 0; i < CHUNK; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const bool live = s + i < end;
                    float gate = float(g[i].v[j]), value = float(v[i].v[j]), u, k;
                    // What the two forms have in common is not to be taken before the branch: it would be held there.
                    if (decltype(far)::value) asm("" : "+v"(gate), "+v"(value));
                    gates(gate, u, k);
                    if (decltype(far)::value) far_gates(gate, u, k);
                    const float add = added(k, value);
                    step(j, live ? u : 1.0f, live ? add : 0.0f);
                }
        };
        if (any_far(most)) steps(std::true_type{});
        else steps(std::false_type{});
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (!GRAD && A[j] == 0.0f && low[j] > 0.0f) A[j] = SMALLEST;
        maps[wave][0][lane * V + j] = A[j];
        maps[wave][1][lane * V + j] = S[j];
    }
    __syncthreads();
    if (wave || !p.inside) return;
    for (int n = 1; n < waves; ++n) {
        const int w = GRAD ? waves - 1 - n : n;
        if (GRAD && n == 1)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                A[j] = maps[waves - 1][0][lane * V + j];
                S[j] = maps[waves - 1][1][lane * V + j];
            }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            A[j] = joined(A[j], maps[w][0][lane * V + j]);
            S[j] = fmaf(maps[w][0][lane * V + j], S[j], maps[w][1][lane * V + j]);
        }
    }
    float *part = a.parts + ((p.segment * a.all + p.b) * 2) * a.width + p.channel;
#pragma unroll
    for (int j = 0; j < V; ++j) part[j] = A[j], part[a.width + j] = S[j];
}

// Segments along the steps, where the channels alone give too few workgroups. They cost another pass over the
// input and another launch: in tenths of a microsecond an unsplit workgroup takes 30 and 27 for 128 steps, whatever
// the others do, split ones 90 and their bytes (BF16, 8 x 1000 x 1024: 26 us unsplit, 28 split; 12 x
// 600 x 1024 18 and 28; 4 x 1000 x 1024 23 and 19; 1 x 1000 x 512 22 and 14).
struct Split {
    i64 segments = 1, segment;
    Split(i64 steps, i64 batch, i64 width) : segment((steps + SPAN - 1) / SPAN * SPAN) {
        const i64 columns = batch * ((width + 63) / 64), spans = segment / SPAN;
        const double states = double(steps) * double(batch) * double(width);
        if (columns >= 256 || spans < 3 || double(30 + 27 * spans) <= 90.0 + states / 45000.0) return;
        const i64 wanted = std::min<i64>((512 + columns - 1) / columns, spans);
        segment = (spans + wanted - 1) / wanted * SPAN;
        segments = (steps + segment - 1) / segment;
    }
    i64 bytes(i64 batch, i64 width) const {
        return segments > 1 ? segments * batch * width * 2 * i64(sizeof(float)) : 0;
    }
};

constexpr i64 MOST_STEPS = i64(1) << 31, MOST_WIDTH = i64(1) << 24, MOST_BATCH = i64(1) << 31;

int check_recurrence(const void *x, int32_t type, i64 steps, i64 batch, i64 width, i64 xt, i64 xb) {
    if (!x || !known_type(type) || steps < 1 || batch < 1 || width < 1 || xt < 0 || xb < 0)
        return fail(MF_E_INVALID, "invalid recurrence arguments");
    if (steps >= MOST_STEPS || width > MOST_WIDTH || batch >= MOST_BATCH)
        return fail(MF_E_UNSUPPORTED, "recurrence of %lld steps, %lld sequences, %lld channels",
                    (long long)steps, (long long)batch, (long long)width);
    if (!aligned(x, type_bytes(type)))
        return fail(MF_E_INVALID, "recurrence input is not aligned to its type");
    return MF_OK;
}

// Calls f(V) with the channels of a lane that reduces segments: two where every row allows it.
template <typename F> int with_group(bool pairs, F f) {
    return pairs ? f(std::integral_constant<int, 2>{}) : f(std::integral_constant<int, 1>{});
}

// Launches kernel over (tiles, sequences, segments), a part of the sequences at a time: a launch has
// fewer than 2^32 threads.
template <typename K>
int launch_recurrence(const char *what, K kernel, RecurrenceArgs a, i64 batch, int v, int waves,
                      hipStream_t s) {
    a.all = batch;
    a.tiles = (a.width + 64 * v - 1) / (64 * v);
    const i64 most = std::max<i64>(1, (i64(1) << 21) / (a.tiles * a.segments));
    for (a.first = 0; a.first < batch; a.first += most) {
        a.batch = std::min(most, batch - a.first);
        hipLaunchKernelGGL(kernel, dim3(u32(a.tiles * a.batch * a.segments)), dim3(64 * waves), 0, s, a);
        const int status = check_launch(what);
        if (status) return status;
    }
    return MF_OK;
}

}  // namespace mf

using namespace mf;

extern "C" {

int mf_recurrence_sizes(int64_t steps, int64_t batch, int64_t width, int64_t *marks, int64_t *workspace) {
    if (steps < 1 || batch < 1 || width < 1 || steps >= MOST_STEPS || width > MOST_WIDTH ||
        batch >= MOST_BATCH || !marks || !workspace)
        return fail(MF_E_INVALID, "invalid recurrence sizes");
    *marks = (steps + SPAN - 1) / SPAN * batch * width * i64(sizeof(float));
    *workspace = Split(steps, batch, width).bytes(batch, width);
    return MF_OK;
}

int mf_recurrence(const void *x, int32_t type, int64_t steps, int64_t batch, int64_t width, int64_t xt,
                  int64_t xb, const float *state, const int64_t *lengths, int32_t reverse, int32_t tanh,
                  void *y, int64_t yt, int64_t yb, float *last, float *marks, void *workspace,
                  int64_t bytes, void *stream) {
    const int status = check_recurrence(x, type, steps, batch, width, xt, xb);
    if (status) return status;
    if (!y || !last || yt < 0 || yb < 0 || !aligned(y, type_bytes(type)) || !aligned(state, 4) ||
        !aligned(lengths, 8) || !aligned(last, 4) || !aligned(marks, 4) || !aligned(workspace, 8))
        return fail(MF_E_INVALID, "invalid recurrence operands");
    const Split split(steps, batch, width);
    if (bytes < split.bytes(batch, width) || (split.segments > 1 && !workspace))
        return fail(MF_E_INVALID, "recurrence workspace of %lld bytes", (long long)bytes);
    RecurrenceArgs a{};
    a.x = x, a.xt = xt, a.xb = xb, a.state = state, a.lengths = lengths;
    a.steps = steps, a.width = width, a.reverse = reverse != 0;
    a.y = y, a.yt = yt, a.yb = yb, a.last = last, a.marks = marks;
    a.segments = split.segments, a.segment = split.segment;
    a.parts = static_cast<float *>(workspace);
    const uintptr_t pair = 2 * type_bytes(type);
    const bool pairs = !((xt | xb | yt | yb | width) & 1) && aligned(x, pair) && aligned(y, pair);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        if (a.segments > 1) {
            const int parts = with_group(pairs, [&](auto group) {
                constexpr int V = decltype(group)::value;
                return launch_recurrence("recurrence parts",
                                         tanh ? k_recurrence_parts<T, V, true, false>
                                              : k_recurrence_parts<T, V, false, false>,
                                         a, batch, V, MOST_WAVES, s);
            });
            if (parts) return parts;
        }
        if (steps > SPAN)
            return launch_recurrence("recurrence", tanh ? k_recurrence<T, true, 8, 16>
                                                        : k_recurrence<T, false, 8, 16>, a, batch, 1, 8, s);
        return launch_recurrence("recurrence", tanh ? k_recurrence<T, true, 16, 8>
                                                    : k_recurrence<T, false, 16, 8>,
                                 a, batch, 1, int((steps + 7) / 8), s);
    });
}

int mf_recurrence_grad(const void *x, int32_t type, int64_t steps, int64_t batch, int64_t width,
                       int64_t xt, int64_t xb, const int64_t *lengths, int32_t reverse, int32_t tanh,
                       const float *marks, const void *dy, int64_t yt, int64_t yb, const float *dlast,
                       void *dx, int64_t dt, int64_t db, float *dstate, void *workspace, int64_t bytes,
                       void *stream) {
    const int status = check_recurrence(x, type, steps, batch, width, xt, xb);
    if (status) return status;
    if (!marks || !dx || dt < 0 || db < 0 || yt < 0 || yb < 0 || !aligned(dx, type_bytes(type)) ||
        !aligned(dy, type_bytes(type)) || !aligned(lengths, 8) || !aligned(marks, 4) || !aligned(dlast, 4) ||
        !aligned(dstate, 4) || !aligned(workspace, 8))
        return fail(MF_E_INVALID, "invalid recurrence gradient arguments");
    const Split split(steps, batch, width);
    if (bytes < split.bytes(batch, width) || (split.segments > 1 && !workspace))
        return fail(MF_E_INVALID, "recurrence workspace of %lld bytes", (long long)bytes);
    RecurrenceArgs a{};
    a.x = x, a.xt = xt, a.xb = xb, a.lengths = lengths;
    a.steps = steps, a.width = width, a.reverse = reverse != 0;
    a.y = const_cast<void *>(dy), a.yt = yt, a.yb = yb, a.last = const_cast<float *>(dlast);
    a.marks = const_cast<float *>(marks), a.dx = dx, a.dt = dt, a.db = db, a.dstate = dstate;
    a.segments = split.segments, a.segment = split.segment;
    a.parts = static_cast<float *>(workspace);
    const uintptr_t pair = 2 * type_bytes(type);
    const bool pairs = !((xt | xb | yt | yb | width) & 1) && aligned(x, pair) && aligned(dy, pair);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        if (a.segments > 1) {
            const int parts = with_group(pairs, [&](auto group) {
                constexpr int V = decltype(group)::value;
                return launch_recurrence("recurrence gradient parts", k_recurrence_parts<T, V, false, true>,
                                         a, batch, V, MOST_WAVES, s);
            });
            if (parts) return parts;
        }
        if (steps > SPAN)
            return launch_recurrence("recurrence gradient", tanh ? k_recurrence_grad<T, true, 8, 16>
                                                                 : k_recurrence_grad<T, false, 8, 16>,
                                     a, batch, 1, 8, s);
        return launch_recurrence("recurrence gradient", tanh ? k_recurrence_grad<T, true, 16, 8>
                                                             : k_recurrence_grad<T, false, 16, 8>,
                                 a, batch, 1, int((steps + 7) / 8), s);
    });
}

}  // extern "C"
