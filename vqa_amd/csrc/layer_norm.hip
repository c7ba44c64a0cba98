// Layer norm over the last axis, forward and backward.
//   y = (x - mean) rstd w + b;   with g = dy w and xh = (x - mean) rstd:
//   dx = rstd (g - mean(g) - xh mean(g xh)),  dw = sum over rows of dy xh,  db = sum over rows of dy
// Both directions are bound by HBM: a row is read once into registers (E elements per lane of its team of 64, 256 or 512
// lanes), the mean and then the mean square of the CENTRED values are taken from there - no cancellation between large
// sums - and the result is written from there.  The backward's workgroups walk over rows and keep their share of dw / db
// in registers; one partial row per workgroup is written and summed in a fixed order (no atomics: the same bits every
// time).
#include <algorithm>
#include "seq.h"

namespace {

// Sums of a and b over the team.  The waves of a larger team meet at ONE barrier: two successive sums use the two halves
// of sh, and a wave that writes a half again has passed the barrier behind which the other waves had read it.
template <int TEAM> __device__ __forceinline__ void team_sum2(float& a, float& b, float2 (*sh)[TEAM / 64], int& half) {
    a = wave_sum(a);
    b = wave_sum(b);
    if constexpr (TEAM > 64) {
        float2* s = sh[half];
        half ^= 1;
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = make_float2(a, b);
        __syncthreads();
        a = b = 0.f;
#pragma unroll
        for (int i = 0; i < TEAM / 64; ++i) { a += s[i].x; b += s[i].y; }
    }
}

// A row is NV vectors of V elements a lane and, where V does not divide the width, one more element of its first lanes.
template <typename T, int V, int TEAM, int NV, bool TAIL>
__global__ __launch_bounds__(TEAM == 64 ? 256 : TEAM) void ln_fwd(const T* __restrict__ x, long ldx,
                                                                  const float* __restrict__ w,
                                                                  const float* __restrict__ bias, long rows, int width,
                                                                  float eps, T* __restrict__ y,
                                                                  float* __restrict__ mean, float* __restrict__ rstd) {
    __shared__ float2 sh[2][TEAM / 64];
    int half = 0;
    const int lane = threadIdx.x % TEAM, main = TAIL ? width - width % V : width;
    const bool tail = TAIL && lane < width - main;
    const long row = (long)blockIdx.x * (TEAM == 64 ? 4 : 1) + (TEAM == 64 ? threadIdx.x / 64 : 0);
    if (row >= rows) return;                               // (whole waves; only where a team is one wave)
    Raw<T, V> r[NV];
    Raw<T, 1> rt;
    float sum = 0.f, zero = 0.f;
    rt.zero();
    if (tail) rt.load(x + row * ldx + main + lane);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * TEAM + lane) * V;
        if (c < main) r[i].load(x + row * ldx + c); else r[i].zero();
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) sum += r[i].get(k);
    if (TAIL) sum += rt.get(0);
    team_sum2<TEAM>(sum, zero, sh, half);
    const float mu = sum / width;
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if ((i * TEAM + lane) * V < main) {
#pragma unroll
            for (int k = 0; k < V; ++k) { const float d = r[i].get(k) - mu; sq += d * d; }
        }
    if (tail) sq += (rt.get(0) - mu) * (rt.get(0) - mu);
    team_sum2<TEAM>(sq, zero, sh, half);
    const float rs = 1.f / sqrtf(sq / width + eps);
    if (lane == 0 && mean) { mean[row] = mu; rstd[row] = rs; }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * TEAM + lane) * V;
        if (c < main) {
            Raw<float, V> wv, bv;
            if (w) wv.load(w + c);
            if (bias) bv.load(bias + c);
            Raw<T, V> o;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                float v = (r[i].get(k) - mu) * rs;
                if (w) v *= wv.get(k);
                if (bias) v += bv.get(k);
                o.set(k, v);
            }
            o.store(y + row * width + c);
        }
    }
    if (tail) {
        const int c = main + lane;
        const float v = (rt.get(0) - mu) * rs * (w ? w[c] : 1.f) + (bias ? bias[c] : 0.f);
        rt.set(0, v);
        rt.store(y + row * width + c);
    }
}

template <typename T, int V, int TEAM, int NV, bool TAIL>
__global__ __launch_bounds__(TEAM == 64 ? 256 : TEAM) void ln_bwd(const T* __restrict__ dy, long lddy,
                                                                  const T* __restrict__ x, long ldx,
                                                                  const float* __restrict__ w,
                                                                  const float* __restrict__ mean,
                                                                  const float* __restrict__ rstd, long rows, int width,
                                                                  T* __restrict__ dx, float* __restrict__ part) {
    constexpr int TEAMS = TEAM == 64 ? 4 : 1;
    __shared__ float2 sh[2][TEAM / 64];
    int half = 0;
    const int lane = threadIdx.x % TEAM, team = TEAM == 64 ? threadIdx.x / 64 : 0;
    const int main = TAIL ? width - width % V : width;
    const bool tail = TAIL && lane < width - main;
    float wv[NV][V], aw[NV][V], ab[NV][V], wt = 0.f, awt = 0.f, abt = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int c = (i * TEAM + lane) * V + k;
            wv[i][k] = c < main ? (w ? w[c] : 1.f) : 0.f;
            aw[i][k] = ab[i][k] = 0.f;
        }
    if (tail) wt = w ? w[main + lane] : 1.f;
    const float inv = 1.f / width;
    const long step = (long)gridDim.x * TEAMS;
    long row = (long)blockIdx.x * TEAMS + team;
    Raw<T, V> xr[NV], gr[NV], xn[NV], gn[NV];
    Raw<T, 1> xt, gt, xnt, gnt;
    float mu = 0.f, rs = 0.f, mun = 0.f, rsn = 0.f;
    // The next row is in flight while this one is worked on.  The loads are straight-line code - a lane past the end loads
    // the last columns again, whose dy it takes as 0, and past the last row that row - because behind a branch that may
    // skip them the compiler waits for the new loads where it needs the old ones.  (A weight of 0 alone does not do: 0
    // times an infinite dy would make NaN of a row whose sums are infinite.)
    auto fetch = [&](long at) {
        at = min(at, rows - 1);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = min((i * TEAM + lane) * V, main - V);
            xn[i].load(x + at * ldx + c);
            gn[i].load(dy + at * lddy + c);
        }
        if constexpr (TAIL) {
            const int c = min(main + lane, width - 1);
            xnt.load(x + at * ldx + c);
            gnt.load(dy + at * lddy + c);
        }
        mun = mean[at];
        rsn = rstd[at];
    };
    fetch(row);
    for (; row < rows; row += step) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            xr[i] = xn[i];
            gr[i] = gn[i];
            if ((i * TEAM + lane) * V >= main) gr[i].zero();
        }
        if (TAIL) {
            xt = xnt;
            gt = gnt;
            if (!tail) gt.zero();
        }
        mu = mun;
        rs = rsn;
        fetch(row + step);
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float xh = (xr[i].get(k) - mu) * rs, d = gr[i].get(k), g = d * wv[i][k];
                s1 += g;
                s2 += g * xh;
                aw[i][k] += d * xh;
                ab[i][k] += d;
            }
        if (TAIL) {
            const float xh = (xt.get(0) - mu) * rs, d = gt.get(0), g = d * wt;
            s1 += g;
            s2 += g * xh;
            awt += d * xh;
            abt += d;
        }
        team_sum2<TEAM>(s1, s2, sh, half);
        s1 *= inv;
        s2 *= inv;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * TEAM + lane) * V;
            if (c < main) {
                Raw<T, V> o;
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const float xh = (xr[i].get(k) - mu) * rs;
                    o.set(k, rs * (gr[i].get(k) * wv[i][k] - s1 - xh * s2));
                }
                o.store(dx + row * width + c);
            }
        }
        if (tail) {
            xt.set(0, rs * (gt.get(0) * wt - s1 - (xt.get(0) - mu) * rs * s2));
            xt.store(dx + row * width + main + lane);
        }
    }
    // the workgroup's share of dw and db: part[blockIdx][2][width]; the four one-wave teams are joined through LDS
    float* out = part + (long)blockIdx.x * 2 * width;
    if constexpr (TEAMS == 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const int c = (i * TEAM + lane) * V + k;
                if (c < main) { out[c] = aw[i][k]; out[width + c] = ab[i][k]; }
            }
        if (tail) { out[main + lane] = awt; out[width + main + lane] = abt; }
    } else {
        constexpr int E = NV * V;
        __shared__ float acc[2 * E * 64], acct[2][8];
        for (int t = 0; t < TEAMS; ++t) {
            if (team == t) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        float* a = acc + (i * V + k) * 64 + lane;
                        a[0] = (t ? a[0] : 0.f) + aw[i][k];
                        a[E * 64] = (t ? a[E * 64] : 0.f) + ab[i][k];
                    }
                if (tail) {
                    acct[0][lane] = (t ? acct[0][lane] : 0.f) + awt;
                    acct[1][lane] = (t ? acct[1][lane] : 0.f) + abt;
                }
            }
            __syncthreads();
        }
        for (int j = threadIdx.x; j < 2 * E * 64; j += 256) {
            const int half_at = j / (E * 64), e = (j / 64) % E, l = j & 63, c = ((e / V) * 64 + l) * V + e % V;
            if (c < main) out[half_at * width + c] = acc[j];
        }
        if (TAIL && team < 2 && tail) out[team * width + main + lane] = acct[team][lane];
    }
}

// Lanes per row and elements per lane.  A wave holds up to 2048 columns, 32 a lane, where its registers allow two waves a
// SIMD: 16-bit rows in the forward, and in the backward where they have no tail (65536 x 2048 bf16: forward 104 us, backward
// 163; with 256 lanes a row 120 and 166).  Else (`wide`) those rows take 256 lanes (backward, 16000 x 1999 bf16: 44 us, 49 with
// one wave; 16000 x 1600 f32: 50 and 59).
struct Shape { int team, e; };
Shape shape_of(int width, bool wide) {
    if (width <= 512) return {64, 8};
    if (width <= 1024) return {64, 16};
    if (width <= 2048) return wide ? Shape{256, 8} : Shape{64, 32};
    if (width <= 4096) return {256, 16};
    return {512, 16};
}
constexpr int MAX_WIDTH = 8192;
constexpr long MAX_ROWS = 1 << 22;                         // of one launch: a grid has fewer than 2^32 threads

int bwd_groups(long rows, int team) {
    const long per = team == 64 ? 4 : 1;
    const long g = (rows + per * 4 - 1) / (per * 4);       // four rows a team, so that the partial rows stay few
    return (int)(g < 1 ? 1 : g > 512 ? 512 : g);
}

template <typename T, int V, bool TAIL, typename F> int by_shape(int width, F f) {
    constexpr bool wide = F::wide(sizeof(T), TAIL);
    const Shape s = shape_of(width - width % V, wide);
    if (s.team == 64 && s.e == 8) return f.template operator()<T, V, 64, 8 / V, TAIL>();
    if (s.team == 64 && s.e == 16) return f.template operator()<T, V, 64, 16 / V, TAIL>();
    if constexpr (wide) {
        if (s.team == 256 && s.e == 8) return f.template operator()<T, V, 256, 8 / V, TAIL>();
    } else {
        if (s.team == 64) return f.template operator()<T, V, 64, 32 / V, TAIL>();
    }
    if (s.team == 256) return f.template operator()<T, V, 256, 16 / V, TAIL>();
    return f.template operator()<T, V, 512, 16 / V, TAIL>();
}
template <typename T, typename F> int by_tail(int width, F f) {
    constexpr int V = 16 / sizeof(T);
    if (width < V) return f.template operator()<T, 1, 64, 8, false>();
    return width % V ? by_shape<T, V, true>(width, f) : by_shape<T, V, false>(width, f);
}
template <typename F> int by_type(int dtype, int width, F f) {
    if (dtype == VQA_F32) return by_tail<float>(width, f);
    if (dtype == VQA_BF16) return by_tail<bf16>(width, f);
    return by_tail<_Float16>(width, f);
}

struct Fwd {
    static constexpr bool wide(int bytes, bool) { return bytes == 4; }
    hipStream_t st; const void* x; long ldx; const float *w, *b; long rows; int width; float eps; void* y; float *mean, *rstd;
    template <typename T, int V, int TEAM, int NV, bool TAIL> int operator()() const {
        for (long r = 0; r < rows; r += MAX_ROWS) {
            const long n = std::min(rows - r, MAX_ROWS), grid = TEAM == 64 ? (n + 3) / 4 : n;
            ln_fwd<T, V, TEAM, NV, TAIL><<<(unsigned)grid, TEAM == 64 ? 256 : TEAM, 0, st>>>(
                static_cast<const T*>(x) + r * ldx, ldx, w, b, n, width, eps, static_cast<T*>(y) + r * width,
                mean ? mean + r : nullptr, rstd ? rstd + r : nullptr);
            CHECK_LAUNCH();
        }
        return VQA_OK;
    }
};
struct Bwd {
    static constexpr bool wide(int bytes, bool tail) { return bytes == 4 || tail; }
    hipStream_t st; const void* dy; long lddy; const void* x; long ldx; const float *w, *mean, *rstd; long rows; int width;
    void* dx; float *dw, *db, *part;
    template <typename T, int V, int TEAM, int NV, bool TAIL> int operator()() const {
        ln_bwd<T, V, TEAM, NV, TAIL><<<bwd_groups(rows, TEAM), TEAM == 64 ? 256 : TEAM, 0, st>>>(
            static_cast<const T*>(dy), lddy, static_cast<const T*>(x), ldx, w, mean, rstd, rows, width,
            static_cast<T*>(dx), part);
        CHECK_LAUNCH();
        if (dw || db) {
            seq_sum_columns(st, part, bwd_groups(rows, TEAM), 2L * width, dw, width, db);
            CHECK_LAUNCH();
        }
        return VQA_OK;
    }
};

bool bad_shape(int dtype, long rows, int width) {
    return !vqa_dtype_ok(dtype) || rows < 1 || rows > 0x7fffffffL || width < 1 || width > MAX_WIDTH;
}

}  // namespace

extern "C" int vqa_layer_norm_fwd(void* stream, int dtype, const void* x, long ldx, const float* weight,
                                  const float* bias, long rows, int width, float eps, void* y, float* stats) {
    if (bad_shape(dtype, rows, width) || !x || !y) return VQA_ERR_ARG;
    return by_type(dtype, width,
                   Fwd{static_cast<hipStream_t>(stream), x, ldx, weight, bias, rows, width, eps, y, stats,
                       stats ? stats + rows : nullptr});
}

extern "C" int vqa_layer_norm_bwd_part(long rows, int width) {
    return rows < 1 || width < 1 || width > MAX_WIDTH ? 0 : bwd_groups(rows, 256);      // (the larger of the two)
}

extern "C" int vqa_layer_norm_bwd(void* stream, int dtype, const void* dy, long lddy, const void* x, long ldx,
                                  const float* weight, const float* stats, long rows, int width, void* dx,
                                  float* dweight, float* dbias, float* part) {
    if (bad_shape(dtype, rows, width) || !dy || !x || !stats || !dx || !part) return VQA_ERR_ARG;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return by_type(dtype, width, Bwd{st, dy, lddy, x, ldx, weight, stats, stats + rows, rows, width, dx, dweight, dbias, part});
}
