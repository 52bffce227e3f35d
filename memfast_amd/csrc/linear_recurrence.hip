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

// A wave takes 64 * V channels and CHUNK steps of them, the up to MOST_WAVES waves of a workgroup
// consecutive chunks: SPAN steps at a time, whose maps they exchange in LDS.
constexpr int CHUNK = 8, MOST_WAVES = 16, SPAN = CHUNK * MOST_WAVES;
constexpr float LOG2E = 1.44269504f, LOG2E_LOW = 1.92596299e-8f, LN2 = 0.693147181f;

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

// exp(-x) for x >= 0: the rounding of x log2(e) is made good, so that far gates keep their digits too.
__device__ __forceinline__ float decay(float x) {
    const float t = -x * LOG2E;
    const float rest = fmaf(-x, LOG2E, -t) - x * LOG2E_LOW;
    const float e = __builtin_amdgcn_exp2f(t);
    return x < 126.0f ? fmaf(e, rest * LN2, e) : e;
}

// sigmoid(g) and sigmoid(-g): the smaller one is not a difference, so either end keeps its digits.
__device__ __forceinline__ void gates(float g, float &u, float &k) {
    const float e = decay(fabsf(g)), big = __builtin_amdgcn_rcpf(1.0f + e), small = e * big;
    u = g >= 0.0f ? big : small;
    k = g >= 0.0f ? small : big;
}

// tanh: (1 - e) / (1 + e) with e = exp(-2 |x|), and where that difference would lose digits the series
// x - x^3 / 3 + 2 x^5 / 15 - 17 x^7 / 315 + 62 x^9 / 2835 (below 1/4 the next term is under 1e-8 of it).
__device__ __forceinline__ float hyperbolic_tangent(float x) {
    const float e = decay(2.0f * fabsf(x));
    const float far = copysignf((1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e), x);
    const float s = x * x;
    float p = fmaf(s, 62.0f / 2835.0f, -17.0f / 315.0f);
    p = fmaf(s, p, 2.0f / 15.0f);
    p = fmaf(s, p, -1.0f / 3.0f);
    return fabsf(x) < 0.25f ? fmaf(x * s, p, x) : far;
}

// What one workgroup works on.
template <typename T, int V> struct Place {
    i64 b, channel, segment, length, begin, end, step;
    bool inside;
    const T *x;

    __device__ __forceinline__ explicit Place(const RecurrenceArgs &a) {
        u32 id = blockIdx.x;
        const u32 tile = id % u32(a.tiles);
        id /= u32(a.tiles);
        b = a.first + id % u32(a.batch);
        segment = id / u32(a.batch);
        const i64 c = (i64(tile) * 64 + (threadIdx.x & 63)) * V;
        inside = c < a.width;
        channel = inside ? c : 0;
        length = a.steps;
        if (a.lengths) {
            length = a.lengths[b];
            length = length < 0 ? 0 : length > a.steps ? a.steps : length;
        }
        begin = segment * a.segment;
        end = min(begin + a.segment, a.steps);
        // Step s of the recurrence lies at time s, or in reverse at length - 1 - s.
        step = a.reverse ? -a.xt : a.xt;
        x = static_cast<const T *>(a.x) + b * a.xb + channel + (a.reverse ? (length - 1) * a.xt : 0);
    }
    __device__ __forceinline__ i64 time(const RecurrenceArgs &a, i64 s) const {
        return a.reverse ? length - 1 - s : s;
    }
    __device__ __forceinline__ i64 at(const RecurrenceArgs &a) const { return b * a.width + channel; }
};

// Gates and candidates of CHUNK steps from s on. Steps past the last are read as the last one, which
// exists (length > 0), and left out later.
template <typename T, int V> struct Loaded {
    Group<T, V> g[CHUNK], v[CHUNK];
    __device__ __forceinline__ void load(const RecurrenceArgs &a, const Place<T, V> &p, i64 s) {
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) {
            const T *row = p.x + min(s + i, p.length - 1) * p.step;
            g[i] = *reinterpret_cast<const Group<T, V> *>(row);
            v[i] = *reinterpret_cast<const Group<T, V> *>(row + a.width);
        }
    }
};

// carry through the maps of the segments first .. last - 1, in order (BACK: from the last on): every
// wave composes its share, whose loads it has under way together, and the shares meet in LDS.
template <int V, bool BACK>
__device__ __forceinline__ void fold(const RecurrenceArgs &a, i64 b, i64 channel, i64 first, i64 last,
                                     float (*maps)[2][64 * V], float (&carry)[V]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
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
                A[j] *= live ? pa[i][j] : 1.0f;
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

// Writes zeros at the times from the sequence's length on.
template <typename T, int V>
__device__ __forceinline__ void blank(const RecurrenceArgs &a, const Place<T, V> &p, T *rows, i64 step,
                                      int wave, int waves, i64 second) {
    if (!p.inside) return;
    const Group<T, V> zero{};
    for (i64 t = max(p.begin, p.length) + wave; t < p.end; t += waves) {
        *reinterpret_cast<Group<T, V> *>(rows + t * step) = zero;
        if (second) *reinterpret_cast<Group<T, V> *>(rows + t * step + second) = zero;
    }
}

template <typename T, int V, bool TANH>
__global__ __launch_bounds__(64 * MOST_WAVES) void k_recurrence(const RecurrenceArgs a) {
    __shared__ float maps[2][MOST_WAVES][2][64 * V];
    const Place<T, V> p(a);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int span = waves * CHUNK;
    T *y = static_cast<T *>(a.y) + p.b * a.yb + p.channel;
    const i64 end = min(p.end, p.length);

    Loaded<T, V> next;
    if (p.begin < end) next.load(a, p, p.begin + wave * CHUNK);
    float carry[V];
#pragma unroll
    for (int j = 0; j < V; ++j) carry[j] = a.state ? a.state[p.at(a) + j] : 0.0f;
    // The state before this segment: the maps of those before it, in order.
    if (p.segment) fold<V, false>(a, p.b, p.channel, 0, p.segment, maps[0], carry);

    int turn = 0;
    for (i64 base = p.begin; base < end; base += span, turn ^= 1) {
        const i64 s = base + wave * CHUNK;
        float u[CHUNK][V], in[CHUNK][V], A[V], S[V];
#pragma unroll
        for (int j = 0; j < V; ++j) A[j] = 1.0f, S[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < CHUNK; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float k, c = float(next.v[i].v[j]);
                gates(float(next.g[i].v[j]), u[i][j], k);
                if (TANH) c = hyperbolic_tangent(c);
                const bool live = s + i < p.length;
                u[i][j] = live ? u[i][j] : 1.0f;
                in[i][j] = live ? k * c : 0.0f;
                A[j] *= u[i][j];
                S[j] = fmaf(u[i][j], S[j], in[i][j]);
            }
        if (base + span < end) next.load(a, p, s + span);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            maps[turn][wave][0][lane * V + j] = A[j];
            maps[turn][wave][1][lane * V + j] = S[j];
        }
        __syncthreads();    // one a turn: the other turn's maps are read before its barrier
        float h[V];
        for (int w = 0; w < waves; ++w) {
            if (w == wave)
#pragma unroll
                for (int j = 0; j < V; ++j) h[j] = carry[j];
#pragma unroll
            for (int j = 0; j < V; ++j)
                carry[j] = fmaf(maps[turn][w][0][lane * V + j], carry[j],
                                maps[turn][w][1][lane * V + j]);
        }
        if (a.marks && wave == 0 && p.inside) {
            float *mark = a.marks + (base / SPAN * a.all) * a.width + p.at(a);
#pragma unroll
            for (int j = 0; j < V; ++j) mark[j] = h[j];
        }
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) {
            Group<T, V> row;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                h[j] = fmaf(u[i][j], h[j], in[i][j]);
                row.v[j] = rounded<T>(h[j]);
            }
            if (p.inside && s + i < p.length)
                *reinterpret_cast<Group<T, V> *>(y + p.time(a, s + i) * a.yt) = row;
        }
    }
    blank(a, p, y, a.yt, wave, waves, 0);
    if (wave == 0 && p.inside && p.segment == a.segments - 1)
#pragma unroll
        for (int j = 0; j < V; ++j) a.last[p.at(a) + j] = carry[j];
}

template <typename T, int V, bool TANH>
__global__ __launch_bounds__(64 * MOST_WAVES) void k_recurrence_grad(const RecurrenceArgs a) {
    __shared__ float maps[2][MOST_WAVES][3][64 * V];
    const Place<T, V> p(a);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int span = waves * CHUNK;
    const T *dy = static_cast<const T *>(a.y) + p.b * a.yb + p.channel;
    T *dx = static_cast<T *>(a.dx) + p.b * a.db + p.channel;
    const i64 end = min(p.end, p.length);

    Loaded<T, V> next;
    Group<T, V> next_dy[CHUNK];
    float mark[V];
    const auto load = [&](i64 base) {
        const i64 s = base + wave * CHUNK;
        next.load(a, p, s);
#pragma unroll
        for (int i = 0; i < CHUNK; ++i)
            next_dy[i] = a.y ? *reinterpret_cast<const Group<T, V> *>(
                                   dy + p.time(a, min(s + i, p.length - 1)) * a.yt)
                             : Group<T, V>{};
#pragma unroll
        for (int j = 0; j < V; ++j)
            mark[j] = a.marks[(base / SPAN * a.all) * a.width + p.at(a) + j];
    };
    const i64 top = p.begin + (end - p.begin - 1) / span * span;
    if (p.begin < end) load(top);
    // The gradient of the state after this segment: the maps of those behind it, from the last on.
    float carry[V];
#pragma unroll
    for (int j = 0; j < V; ++j) carry[j] = a.last ? a.last[p.at(a) + j] : 0.0f;
    if (p.segment + 1 < a.segments)
        fold<V, true>(a, p.b, p.channel, p.segment + 1, a.segments,
                      reinterpret_cast<float (*)[2][64 * V]>(&maps), carry);

    int turn = 0;
    if (p.begin < end)
        for (i64 base = top; base >= p.begin; base -= span, turn ^= 1) {
            const i64 s = base + wave * CHUNK;
            float u[CHUNK][V], k[CHUNK][V], c[CHUNK][V], g[CHUNK][V], A[V], S[V], Q[V], h[V], r[V];
#pragma unroll
            for (int j = 0; j < V; ++j) A[j] = 1.0f, S[j] = 0.0f, Q[j] = 0.0f, h[j] = mark[j];
#pragma unroll
            for (int i = 0; i < CHUNK; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    gates(float(next.g[i].v[j]), u[i][j], k[i][j]);
                    c[i][j] = float(next.v[i].v[j]);
                    if (TANH) c[i][j] = hyperbolic_tangent(c[i][j]);
                    const bool live = s + i < p.length;
                    u[i][j] = live ? u[i][j] : 1.0f;
                    k[i][j] = live ? k[i][j] : 0.0f;
                    c[i][j] = live ? c[i][j] : 0.0f;
                    g[i][j] = live ? float(next_dy[i].v[j]) : 0.0f;
                    A[j] *= u[i][j];
                    S[j] = fmaf(u[i][j], S[j], k[i][j] * c[i][j]);
                }
#pragma unroll
            for (int i = CHUNK - 1; i >= 0; --i)
#pragma unroll
                for (int j = 0; j < V; ++j) Q[j] = u[i][j] * (g[i][j] + Q[j]);
            if (base > p.begin) load(base - span);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                maps[turn][wave][0][lane * V + j] = A[j];
                maps[turn][wave][1][lane * V + j] = S[j];
                maps[turn][wave][2][lane * V + j] = Q[j];
            }
            __syncthreads();
            for (int w = 0; w < wave; ++w)
#pragma unroll
                for (int j = 0; j < V; ++j)
                    h[j] = fmaf(maps[turn][w][0][lane * V + j], h[j], maps[turn][w][1][lane * V + j]);
            for (int w = waves - 1; w >= 0; --w) {
                if (w == wave)
#pragma unroll
                    for (int j = 0; j < V; ++j) r[j] = carry[j];
#pragma unroll
                for (int j = 0; j < V; ++j)
                    carry[j] = fmaf(maps[turn][w][0][lane * V + j], carry[j],
                                    maps[turn][w][2][lane * V + j]);
            }
            // Factors of G in both gradients, then G from the last step back.
#pragma unroll
            for (int i = 0; i < CHUNK; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float before = h[j];
                    h[j] = fmaf(u[i][j], before, k[i][j] * c[i][j]);
                    const float dv = TANH ? k[i][j] * fmaf(-c[i][j], c[i][j], 1.0f) : k[i][j];
                    c[i][j] = (before - c[i][j]) * (u[i][j] * k[i][j]);
                    k[i][j] = dv;
                }
#pragma unroll
            for (int i = CHUNK - 1; i >= 0; --i) {
                Group<T, V> dg, dv;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float G = g[i][j] + r[j];
                    dg.v[j] = rounded<T>(G * c[i][j]);
                    dv.v[j] = rounded<T>(G * k[i][j]);
                    r[j] = u[i][j] * G;
                }
                if (p.inside && s + i < p.length) {
                    T *row = dx + p.time(a, s + i) * a.dt;
                    *reinterpret_cast<Group<T, V> *>(row) = dg;
                    *reinterpret_cast<Group<T, V> *>(row + a.width) = dv;
                }
            }
        }
    blank(a, p, dx, a.dt, wave, waves, a.width);
    if (a.dstate && wave == 0 && p.inside && p.segment == 0)
#pragma unroll
        for (int j = 0; j < V; ++j) a.dstate[p.at(a) + j] = carry[j];
}

// A and S of every segment but the last (GRAD: A and Q of every segment but the first), each wave its
// share of the segment's steps.
template <typename T, int V, bool TANH, bool GRAD>
__global__ __launch_bounds__(64 * MOST_WAVES) void k_recurrence_parts(const RecurrenceArgs a) {
    __shared__ float maps[MOST_WAVES][2][64 * V];
    Place<T, V> p(a);
    if (p.segment == (GRAD ? 0 : a.segments - 1)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const T *dy = static_cast<const T *>(a.y) + p.b * a.yb + p.channel;
    const i64 share = a.segment / waves, end = min(p.begin + (wave + 1) * share, p.length);
    float A[V], S[V];
#pragma unroll
    for (int j = 0; j < V; ++j) A[j] = 1.0f, S[j] = 0.0f;
    for (i64 s = p.begin + wave * share; s < end; s += CHUNK) {
        Group<T, V> g[CHUNK], v[CHUNK];
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) {
            const i64 at = min(s + i, p.length - 1);
            const T *row = p.x + at * p.step;
            g[i] = *reinterpret_cast<const Group<T, V> *>(row);
            if (!GRAD) v[i] = *reinterpret_cast<const Group<T, V> *>(row + a.width);
            else v[i] = a.y ? *reinterpret_cast<const Group<T, V> *>(dy + p.time(a, at) * a.yt)
                            : Group<T, V>{};
        }
#pragma unroll
        for (int i = 0; i < CHUNK; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const bool live = s + i < end;
                float u, k, c = float(v[i].v[j]);
                gates(float(g[i].v[j]), u, k);
                u = live ? u : 1.0f;
                if (GRAD) {     // r -> A u (dy + r) + S
                    A[j] *= u;
                    S[j] = fmaf(A[j], live ? c : 0.0f, S[j]);
                } else {
                    if (TANH) c = hyperbolic_tangent(c);
                    A[j] *= u;
                    S[j] = fmaf(u, S[j], live ? k * c : 0.0f);
                }
            }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
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
            A[j] *= maps[w][0][lane * V + j];
            S[j] = fmaf(maps[w][0][lane * V + j], S[j], maps[w][1][lane * V + j]);
        }
    }
    float *part = a.parts + ((p.segment * a.all + p.b) * 2) * a.width + p.channel;
#pragma unroll
    for (int j = 0; j < V; ++j) part[j] = A[j], part[a.width + j] = S[j];
}

// Segments along the steps: where the channels alone give too few workgroups, and there are steps
// enough for each to be SPAN of them at least.
struct Split {
    i64 segments = 1, segment;
    Split(i64 steps, i64 batch, i64 width) : segment((steps + SPAN - 1) / SPAN * SPAN) {
        const i64 columns = batch * ((width + 127) / 128), spans = segment / SPAN;
        if (columns >= 256 || spans < 4) return;
        const i64 wanted = std::min<i64>({(512 + columns - 1) / columns, spans / 2, 256});
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

// Calls f(V) with the channels of a lane: two where every row of every tensor allows it.
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

int waves_of(i64 steps) { return int(std::min<i64>(MOST_WAVES, (steps + CHUNK - 1) / CHUNK)); }

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
    if (!y || !last || yt < 0 || yb < 0 || !aligned(y, type_bytes(type)))
        return fail(MF_E_INVALID, "invalid recurrence outputs");
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
        return with_group(pairs, [&](auto group) {
            constexpr int V = decltype(group)::value;
            if (a.segments > 1) {
                const int parts = launch_recurrence(
                    "recurrence parts", tanh ? k_recurrence_parts<T, V, true, false>
                                             : k_recurrence_parts<T, V, false, false>,
                    a, batch, V, MOST_WAVES, s);
                if (parts) return parts;
            }
            return launch_recurrence("recurrence", tanh ? k_recurrence<T, V, true> : k_recurrence<T, V, false>,
                                     a, batch, V, waves_of(steps), s);
        });
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
        !aligned(dy, type_bytes(type)))
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
    const bool pairs = !((xt | xb | yt | yb | dt | db | width) & 1) && aligned(x, pair) &&
                       aligned(dy, pair) && aligned(dx, pair);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        return with_group(pairs, [&](auto group) {
            constexpr int V = decltype(group)::value;
            if (a.segments > 1) {
                const int parts = launch_recurrence(
                    "recurrence gradient parts", tanh ? k_recurrence_parts<T, V, true, true>
                                                      : k_recurrence_parts<T, V, false, true>,
                    a, batch, V, MOST_WAVES, s);
                if (parts) return parts;
            }
            return launch_recurrence("recurrence gradient",
                                     tanh ? k_recurrence_grad<T, V, true> : k_recurrence_grad<T, V, false>,
                                     a, batch, V, waves_of(steps), s);
        });
    });
}

}  // extern "C"
