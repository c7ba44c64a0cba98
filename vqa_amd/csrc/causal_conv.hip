// The short causal convolution over tokens (one filter of 2 to 4 taps per channel), forward, backward and for one token.
//   pre_t = bias + sum_k w[:, k] x_{t - W + 1 + k},  y_t = pre_t or silu(pre_t)
//   g_t = dy_t (silu'(pre_t));  dx_t = sum_k w[:, k] g_{t + W - 1 - k};  dw[:, k] = sum g_t x_{t - W + 1 + k};  db = sum g_t
// Rows before the first are the W - 1 rows of `state` (zeros without one); rows at or past a sequence's length are neither
// read into a sum nor answered (zero rows); the state handed on is the last W - 1 rows before that length.
// All of it is bound by HBM, the backward nearly as much by its 35 operations per element: a thread owns four channels and
// walks down a chunk of rows with the filter's window in registers, so a row is loaded once per chunk, plus W - 1 rows at its
// border.  The backward recomputes pre_t from x (nothing is saved) and carries the window of g the same way.
// Measured at 8 x 4096 x 2048 bf16, 4 taps, silu: forward 56 us = 4.8 TB/s, backward 87 us = 4.6 TB/s (a large copy: 5.1).
#include "seq.h"

namespace {

constexpr int RB = 4;          // rows a forward thread has in flight (8 x 4096 x 2048 bf16: 56 us; with 8 rows, or 8 channels a thread, 64-68:
                               // too few waves fit)

template <typename T, int V, int W, bool SILU>
__global__ __launch_bounds__(256) void conv_fwd(const T* __restrict__ x, long xb, long xl, const float* __restrict__ w,
                                                const float* __restrict__ bias, const T* __restrict__ state,
                                                const int* __restrict__ lengths, int B, int L, int D, int chunk,
                                                T* __restrict__ y, T* __restrict__ last) {
    const int nv = (D + V - 1) / V, nchunk = (L + chunk - 1) / chunk;
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= (long)B * nchunk * nv) return;
    const int c = min((int)(id % nv) * V, D - V);          // (the last vector of an odd width overlaps: twice the same results)
    const int q = (int)(id / nv);
    const int b = q / nchunk, t0 = (q % nchunk) * chunk, t1 = min(L, t0 + chunk);
    const int len = lengths ? max(0, min(L, lengths[b])) : L;
    const T* xr = x + b * xb + c;
    const T* sr = state ? state + (long)b * (W - 1) * D + c : nullptr;
    auto row = [&](int t, Raw<T, V>& r) {                  // row t of the sequence with its past
        r.zero();
        if (t >= 0) { if (t < len) r.load(xr + t * xl); }
        else if (sr) r.load(sr + (long)(t + W - 1) * D);
    };
    float wk[W][V], bv[V], win[W][V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        bv[v] = bias ? bias[c + v] : 0.f;
#pragma unroll
        for (int k = 0; k < W; ++k) wk[k][v] = w[(long)(c + v) * W + k];
    }
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
        Raw<T, V> r;
        row(t0 - (W - 1) + k, r);
#pragma unroll
        for (int v = 0; v < V; ++v) win[k][v] = r.get(v);
    }
    for (int s = t0; s < t1; s += RB) {
        Raw<T, V> r[RB];
#pragma unroll
        for (int i = 0; i < RB; ++i)
            if (s + i < t1) row(s + i, r[i]);
#pragma unroll
        for (int i = 0; i < RB; ++i) {
            if (s + i < t1) {
                Raw<T, V> o;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    win[W - 1][v] = r[i].get(v);
                    float p = bv[v];
#pragma unroll
                    for (int k = 0; k < W; ++k) p += wk[k][v] * win[k][v];
#pragma unroll
                    for (int k = 0; k < W - 1; ++k) win[k][v] = win[k + 1][v];
                    o.set(v, s + i < len ? (SILU ? silu_f(p) : p) : 0.f);
                }
                o.store(y + ((long)b * L + s + i) * D + c);
            }
        }
    }
    if (last && t0 == 0) {
#pragma unroll
        for (int k = 0; k < W - 1; ++k) {
            Raw<T, V> r;
            row(len - (W - 1) + k, r);
            r.store(last + ((long)b * (W - 1) + k) * D + c);
        }
    }
}

// LX lanes across channels, 256 / LX chunks of rows side by side; part[blockIdx.y][W + 1][D].
template <typename T, int V, int W, bool SILU>
__global__ __launch_bounds__(256) void conv_bwd(const T* __restrict__ dy, long gb, long gl, const T* __restrict__ dlast,
                                                const T* __restrict__ x, long xb, long xl, const float* __restrict__ w,
                                                const float* __restrict__ bias, const T* __restrict__ state,
                                                const int* __restrict__ lengths, int B, int L, int D, int chunk, int lx,
                                                T* __restrict__ dx, T* __restrict__ dstate, float* __restrict__ part) {
    __shared__ float acc[256 * V];
    const int nchunk = (L + chunk - 1) / chunk, ly = 256 / lx;
    const int lane = threadIdx.x % lx, team = threadIdx.x / lx;
    const bool on = (blockIdx.x * lx + lane) * V < D;
    const int c = min((int)(blockIdx.x * lx + lane) * V, D - V);      // (as in conv_fwd)
    float wk[W][V], bv[V], aw[W][V], ab[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        bv[v] = on && bias ? bias[c + v] : 0.f;
        ab[v] = 0.f;
#pragma unroll
        for (int k = 0; k < W; ++k) { wk[k][v] = on ? w[(long)(c + v) * W + k] : 0.f; aw[k][v] = 0.f; }
    }
    const int total = on ? B * nchunk : 0;
    for (int q = blockIdx.y * ly + team; q < total; q += gridDim.y * ly) {
        const int b = q / nchunk, t0 = (q % nchunk) * chunk, t1 = min(L, t0 + chunk);
        const int len = lengths ? max(0, min(L, lengths[b])) : L;
        const T* xr = x + b * xb + c;
        const T* gr = dy + b * gb + c;
        const T* sr = state ? state + (long)b * (W - 1) * D + c : nullptr;
        float win[W][V], gw[W][V];                         // x and g of the last W - 1 rows, oldest first
#pragma unroll
        for (int k = 0; k < W - 1; ++k) {
            Raw<T, V> r;
            r.zero();
            const int t = t0 - (W - 1) + k;
            if (t >= 0) { if (t < len) r.load(xr + t * xl); }
            else if (sr) r.load(sr + (long)(t + W - 1) * D);
#pragma unroll
            for (int v = 0; v < V; ++v) { win[k][v] = r.get(v); gw[k][v] = 0.f; }
        }
        // step s takes in g_s and gives out the gradient of row s - (W - 1): the first chunk begins with the state's rows
        const int end = t1 + W - 1;
        auto step = [&](int s, const Raw<T, V>& rx, const Raw<T, V>& rg) {     // one row with every guard
            Raw<T, V> o;
            const int t = s - (W - 1), r = s - len;        // row answered; its place among the rows handed on
            float e[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                win[W - 1][v] = rx.get(v);
                float p = bv[v];
#pragma unroll
                for (int k = 0; k < W; ++k) p += wk[k][v] * win[k][v];
                const float d = rg.get(v);
                gw[W - 1][v] = s < len ? (SILU ? d * dsilu_f(p) : d) : 0.f;
                if (s < t1) {                              // (a row past the chunk is another's to sum)
                    ab[v] += gw[W - 1][v];
#pragma unroll
                    for (int k = 0; k < W; ++k) aw[k][v] += gw[W - 1][v] * win[k][v];
                }
                e[v] = 0.f;
#pragma unroll
                for (int k = 0; k < W; ++k) e[v] += wk[k][v] * gw[W - 1 - k][v];
#pragma unroll
                for (int k = 0; k < W - 1; ++k) { win[k][v] = win[k + 1][v]; gw[k][v] = gw[k + 1][v]; }
            }
            if (dlast && r >= 0 && r < W - 1) {
                Raw<T, V> dl;
                dl.load(dlast + ((long)b * (W - 1) + r) * D + c);
#pragma unroll
                for (int v = 0; v < V; ++v) e[v] += dl.get(v);
            }
#pragma unroll
            for (int v = 0; v < V; ++v) o.set(v, e[v]);
            if (t >= t0) o.store(dx + ((long)b * L + t) * D + c);
            else if (t < 0 && dstate) o.store(dstate + ((long)b * (W - 1) + s) * D + c);
        };
        constexpr int U = W == 3 ? 3 : 4;
        auto some = [&](int from, int to) {                // up to U rows of them, loaded together
            Raw<T, V> rx[U], rg[U];
#pragma unroll
            for (int i = 0; i < U; ++i) {
                rx[i].zero();
                rg[i].zero();
                if (from + i < min(to, len)) { rx[i].load(xr + (from + i) * xl); rg[i].load(gr + (from + i) * gl); }
            }
#pragma unroll
            for (int i = 0; i < U; ++i)
                if (from + i < to) step(from + i, rx[i], rg[i]);
        };
        int s = t0 + W - 1;
        some(t0, s);
        // the body: rows that are the chunk's own, before the sequence's end, and answer one of the chunk's.  U rows at a
        // time, the next U in flight; the windows turn instead of moving (U is a multiple of W)
        const int body = min(t1, len) - U;
        if (s <= body) {
            Raw<T, V> nx[U], ng[U];
#pragma unroll
            for (int i = 0; i < U; ++i) { nx[i].load(xr + (s + i) * xl); ng[i].load(gr + (s + i) * gl); }
            for (; s <= body; s += U) {
                Raw<T, V> rx[U], rg[U];
#pragma unroll
                for (int i = 0; i < U; ++i) { rx[i] = nx[i]; rg[i] = ng[i]; }
                if (s + U <= body) {
#pragma unroll
                    for (int i = 0; i < U; ++i) { nx[i].load(xr + (s + U + i) * xl); ng[i].load(gr + (s + U + i) * gl); }
                }
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    Raw<T, V> o;
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        win[(i + W - 1) % W][v] = rx[i].get(v);
                        float p = bv[v];
#pragma unroll
                        for (int k = 0; k < W; ++k) p += wk[k][v] * win[(i + k) % W][v];
                        const float d = rg[i].get(v), g = SILU ? d * dsilu_f(p) : d;
                        gw[(i + W - 1) % W][v] = g;
                        ab[v] += g;
                        float e = wk[0][v] * g;
#pragma unroll
                        for (int k = 1; k < W; ++k) e += wk[k][v] * gw[(i + W - 1 - k) % W][v];
#pragma unroll
                        for (int k = 0; k < W; ++k) aw[k][v] += g * win[(i + k) % W][v];
                        o.set(v, e);
                    }
                    o.store(dx + ((long)b * L + s + i - (W - 1)) * D + c);
                }
            }
        }
        for (; s < end; s += U) some(s, min(s + U, end));
    }
    // the chunks that this workgroup worked on side by side are joined in a fixed order
    float* out = part + (long)blockIdx.y * (W + 1) * D;
#pragma unroll
    for (int k = 0; k <= W; ++k) {
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v * 256 + threadIdx.x] = k < W ? aw[k < W ? k : 0][v] : ab[v];
        __syncthreads();
        if (team == 0 && on) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float a = 0.f;
                for (int j = 0; j < ly; ++j) a += acc[v * 256 + j * lx + lane];
                out[k < W ? (long)(c + v) * W + k : (long)W * D + c + v] = a;
            }
        }
    }
}

template <typename T, int V, int W, bool SILU>
__global__ __launch_bounds__(256) void conv_token(const T* __restrict__ x, long xb, T* __restrict__ state, long sb,
                                                  long sl, const float* __restrict__ w, const float* __restrict__ bias,
                                                  int B, int D, T* __restrict__ y) {
    const int nv = (D + V - 1) / V;
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= (long)B * nv) return;
    const int c = (int)(id % nv) * V;
    const long b = id / nv;
    Raw<T, V> r[W];
    T* s = state + b * sb + c;
#pragma unroll
    for (int k = 0; k < W - 1; ++k) r[k].load(s + k * sl);
    r[W - 1].load(x + b * xb + c);
    Raw<T, V> o;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float p = bias ? bias[c + v] : 0.f;
#pragma unroll
        for (int k = 0; k < W; ++k) p += w[(long)(c + v) * W + k] * r[k].get(v);
        o.set(v, SILU ? silu_f(p) : p);
    }
    o.store(y + b * D + c);
#pragma unroll
    for (int k = 0; k < W - 1; ++k) r[k + 1].store(s + k * sl);
}

// f(element type, V, taps, silu)
template <typename T, int V, typename F> int by_taps(int taps, int silu, F f) {
    if (taps == 2) return silu ? f.template operator()<T, V, 2, true>() : f.template operator()<T, V, 2, false>();
    if (taps == 3) return silu ? f.template operator()<T, V, 3, true>() : f.template operator()<T, V, 3, false>();
    return silu ? f.template operator()<T, V, 4, true>() : f.template operator()<T, V, 4, false>();
}
template <typename F> int by_type(int dtype, bool vec, int taps, int silu, F f) {
    if (dtype == VQA_F32) return vec ? by_taps<float, 4>(taps, silu, f) : by_taps<float, 1>(taps, silu, f);
    if (dtype == VQA_BF16) return vec ? by_taps<bf16, 4>(taps, silu, f) : by_taps<bf16, 1>(taps, silu, f);
    return vec ? by_taps<_Float16, 4>(taps, silu, f) : by_taps<_Float16, 1>(taps, silu, f);
}

bool bad_shape(int dtype, int B, long L, int D, int taps) {
    return !vqa_dtype_ok(dtype) || B < 1 || L < 1 || D < 1 || taps < 2 || taps > 4 || D > 25000000 ||
           (double)B * L > 1e9 || (double)B * L * D > 4e11 ||
           (double)B * ((L + 31) / 32) * (D < 4 ? D : (D + 3) / 4) > 4e9;       // (a grid has fewer than 2^32 threads)
}

int fwd_chunk(int B, int L, int nv) {
    // rows per thread: long chunks read few border rows again, but 256 CUs want some 256k threads
    int chunk = 32;
    while (chunk > 8 && (long)B * ((L + chunk - 1) / chunk) * nv < 262144) chunk /= 2;
    return chunk;
}

struct Fwd {
    hipStream_t st; const void* x; long xb, xl; const float *w, *bias; const void* state; const int* lengths; int B, L, D;
    void *y, *last;
    template <typename T, int V, int W, bool SILU> int operator()() const {
        const int nv = (D + V - 1) / V, chunk = fwd_chunk(B, L, nv);
        const long n = (long)B * ((L + chunk - 1) / chunk) * nv;
        conv_fwd<T, V, W, SILU><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(
            static_cast<const T*>(x), xb, xl, w, bias, static_cast<const T*>(state), lengths, B, L, D, chunk,
            static_cast<T*>(y), static_cast<T*>(last));
        CHECK_LAUNCH();
        return VQA_OK;
    }
};

// The backward's grid: lx lanes x V channels across, the rest of a workgroup's 256 threads down the chunks of rows.  Chunks as
// long as 100k threads allow (every chunk computes W - 1 rows of its neighbour's g again and steps in and out of the
// body's unrolled rows; while border rows were still loaded one by one, 8 x 4096 x 2048 bf16 took 94 us with 128 rows, 105 with
// 64, 116 with 32); 64 x 256 x 1024 takes 32 us
// where chunks shrink to keep 65k or 100k threads, 44 us where 32k are let through.
struct Grid { int lx, gx, gy, chunk; };
Grid bwd_grid(int B, int L, int D, int V) {
    const int nv = (D + V - 1) / V;
    int lx = 64;                                           // a row's pieces as long as a quarter of idle lanes allows
    while (lx > 8 && (nv + lx - 1) / lx * lx > nv + nv / 4) lx /= 2;
    const int gx = (nv + lx - 1) / lx, ly = 256 / lx;
    int chunk = 128;
    while (chunk > 8 && (long)B * ((L + chunk - 1) / chunk) * gx * lx < 100000) chunk /= 2;
    const long chunks = (long)B * ((L + chunk - 1) / chunk);
    long gy = (chunks + ly - 1) / ly;
    const long most = gx >= 1024 ? 1 : 1024 / gx;
    if (gy > most) gy = most;
    return {lx, gx, (int)gy, chunk};
}
struct Bwd {
    hipStream_t st; const void* dy; long gb, gl; const void* dlast; const void* x; long xb, xl; const float *w, *bias;
    const void* state; const int* lengths; int B, L, D; void *dx, *dstate; float* part;
    template <typename T, int V, int W, bool SILU> int operator()() const {
        const Grid g = bwd_grid(B, L, D, V);
        conv_bwd<T, V, W, SILU><<<dim3(g.gx, g.gy), 256, 0, st>>>(
            static_cast<const T*>(dy), gb, gl, static_cast<const T*>(dlast), static_cast<const T*>(x), xb, xl, w, bias,
            static_cast<const T*>(state), lengths, B, L, D, g.chunk, g.lx, static_cast<T*>(dx), static_cast<T*>(dstate),
            part);
        CHECK_LAUNCH();
        return VQA_OK;
    }
};
struct Token {
    hipStream_t st; const void* x; long xb; void* state; long sb, sl; const float *w, *bias; int B, D; void* y;
    template <typename T, int V, int W, bool SILU> int operator()() const {
        const long n = (long)B * ((D + V - 1) / V);
        conv_token<T, V, W, SILU><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(
            static_cast<const T*>(x), xb, static_cast<T*>(state), sb, sl, w, bias, B, D, static_cast<T*>(y));
        CHECK_LAUNCH();
        return VQA_OK;
    }
};

}  // namespace

extern "C" int vqa_causal_conv_fwd(void* stream, int dtype, const void* x, long x_batch, long x_row, const float* weight,
                                   const float* bias, const void* state, const int* lengths, int B, int L, int D,
                                   int taps, int silu, void* y, void* last) {
    if (bad_shape(dtype, B, L, D, taps) || !x || !weight || !y) return VQA_ERR_ARG;
    return by_type(dtype, D >= 4, taps, silu,
                      Fwd{static_cast<hipStream_t>(stream), x, x_batch, x_row, weight, bias, state, lengths, B, L, D, y, last});
}

extern "C" int vqa_causal_conv_bwd_part(int B, int L, int D) {
    if (bad_shape(VQA_F32, B, L, D, 4)) return 0;
    const int a = bwd_grid(B, L, D, 1).gy, b = bwd_grid(B, L, D, 4).gy;      // either form may be taken
    return a > b ? a : b;
}

extern "C" int vqa_causal_conv_bwd(void* stream, int dtype, const void* dy, long dy_batch, long dy_row, const void* dlast,
                                   const void* x, long x_batch, long x_row, const float* weight, const float* bias,
                                   const void* state, const int* lengths, int B, int L, int D, int taps, int silu,
                                   void* dx, float* dweight, float* dbias, void* dstate, float* part) {
    if (bad_shape(dtype, B, L, D, taps) || !dy || !x || !weight || !dx || !dweight || !part) return VQA_ERR_ARG;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const int rc = by_type(dtype, D >= 4, taps, silu,
                              Bwd{st, dy, dy_batch, dy_row, dlast, x, x_batch, x_row, weight, bias, state, lengths, B, L, D,
                                  dx, dstate, part});
    if (rc != VQA_OK) return rc;
    seq_sum_columns(st, part, bwd_grid(B, L, D, D >= 4 ? 4 : 1).gy, (long)(taps + 1) * D, dweight, (long)taps * D, dbias);
    CHECK_LAUNCH();
    return VQA_OK;
}

extern "C" int vqa_causal_conv_token(void* stream, int dtype, const void* x, long x_batch, void* state, long state_batch,
                                     long state_row, const float* weight, const float* bias, int B, int D, int taps,
                                     int silu, void* y) {
    if (bad_shape(dtype, B, 1, D, taps) || (D % 4 != 0 && (double)B * D > 4e9) || !x || !state || !weight || !y)
        return VQA_ERR_ARG;
    return by_type(dtype, D % 4 == 0, taps, silu,            // (in place: no two threads may take the same channel)
                   Token{static_cast<hipStream_t>(stream), x, x_batch, state, state_batch, state_row, weight, bias, B, D, y});
}
