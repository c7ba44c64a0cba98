// The selective state space scan: forward, backward and for one token.  Per channel d with states n < N (N <= 64):
//   dt_t = softplus(raw_t + dt_bias);  h_t[n] = exp(dt_t a[n]) h_{t-1}[n] + (dt_t x_t) b_t[n]
//   core_t = sum_n c_t[n] h_t[n] + skip x_t;  y_t = core_t silu(gate_t)
// b and c are shared by the channels of a group.  With dcore = dy silu(gate), G_t the gradient of h_t:
//   G_t = dcore_t c_t + exp(dt_{t+1} a) G_{t+1};  th_t = G_t exp(dt_t a) h_{t-1}
//   dx = dt sum_n G b + skip dcore;  draw = (sum_n a th + x sum_n G b) softplus'(raw + dt_bias);  da = sum_t dt th
//   db_t = sum_d G dt x;  dc_t = sum_d h dcore;  dgate = dy core silu'(gate);  dskip = sum dcore x;  ddt_bias = sum draw
// Tokens at or past a sequence's length: dt = 0 (the state stands still), rows and gradients 0; what lies there is never read
// into a sum (selected away, not multiplied by 0).
//
// Arithmetic, not memory, bounds it: N exponentials and 4 N other operations per (token, channel) against 8 bytes.  It
// stays in f32 on the vector ALU (the decay differs per channel AND state, so there is no matrix product in it).  One wave
// works on 16 CH channels: lane = 16 channel lanes x 4 state rows, each lane holding CH channels x NS states (CH NS = 16) in
// registers.  What a token needs per channel (dt, dt x, ...) and per state (b, c) is staged in LDS in f32, TT tokens at a
// time, by a second mapping of the lanes in which global rows are read 16 bytes a lane; the next tile's rows are in flight
// meanwhile.  Sums over states are three lane-swaps, sums over channels DPP adds.
// With few rows the tokens are cut into segments: a first pass finds each segment's own end state and total decay (the
// product of decays is exp(a sum dt)), a small one chains them, and the full pass starts every segment from its true
// state.  The backward does the same from the other end.  For the backward the forward keeps h before every tile.
#include "seq.h"

namespace {

typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));
constexpr int TT = 8;                      // tokens of a tile
constexpr int LANE_STATE = 1024;           // floats of one wave's states: 64 lanes x CH NS
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct Rows { const void* p; long batch, row; };          // [B][L][...], element strides; the last axis is contiguous

struct Args {
    Rows x, dt, gate, b, c, dy;
    const float *a, *skip, *dt_bias, *state, *dlast;
    const int* lengths;
    int softplus, B, L, D, N, G;
    int nblk, segs, seg_len, bgroups;      // waves across a group's channels, segments, tokens per segment, batch groups
    void* y; float* last;
    float *keep, *seg_h, *seg_dt;          // h before every tile; per segment: state, then the true incoming state; sum dt
    void *dx, *ddt, *dgate; float *part_bc, *part_p, *dstate;
};

// The wave's own LDS traffic in program order: the hardware keeps it, this keeps the compiler from moving it.
__device__ __forceinline__ void lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// log(1 + exp(v)) to relative precision on both sides: log1p(e) = 2 atanh(e / (2 + e)) as its series (e <= 1, so the
// argument is at most 1/3 and the next term under 2e-8 of the sum)
__device__ __forceinline__ float softplus_f(float v) {
    const float e = exp_f(-fabsf(v));
    const float s = e * __builtin_amdgcn_rcpf(2.f + e), q = s * s;
    float p = 1.f / 13.f;
    p = p * q + 1.f / 11.f;
    p = p * q + 1.f / 9.f;
    p = p * q + 1.f / 7.f;
    p = p * q + 1.f / 5.f;
    p = p * q + 1.f / 3.f;
    p = p * q + 1.f;
    return fmaxf(v, 0.f) + 2.f * s * p;
}

// v[i]: lane (row r, channel lane) holds its row's share of channel i.  -> the sum over the 4 rows of channel own(r).
template <int CH> __device__ __forceinline__ int own_channel(int r) { return CH == 4 ? r : CH == 2 ? r >> 1 : 0; }
__device__ __forceinline__ float swap_add32(float a, float b) {        // lanes 0-31: a over both halves, 32-63: b
    const u32x2_t s = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(s.x) + __uint_as_float(s.y);
}
__device__ __forceinline__ float swap_add16(float a, float b) {        // even rows: a over the row pair, odd rows: b
    const u32x2_t s = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(s.x) + __uint_as_float(s.y);
}
template <int CH> __device__ __forceinline__ float sum_states(const float (&v)[CH]) {
    if constexpr (CH == 4) return swap_add16(swap_add32(v[0], v[2]), swap_add32(v[1], v[3]));
    else if constexpr (CH == 2) { const float s = swap_add32(v[0], v[1]); return swap_add16(s, s); }
    else { const float s = swap_add32(v[0], v[0]); return swap_add16(s, s); }
}

template <int N> __device__ __forceinline__ void lds_read(const float* p, float (&v)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 t = *reinterpret_cast<const float4*>(p + i);
            v[i] = t.x; v[i + 1] = t.y; v[i + 2] = t.z; v[i + 3] = t.w;
        }
    } else if constexpr (N == 2) {
        const float2 t = *reinterpret_cast<const float2*>(p);
        v[0] = t.x; v[1] = t.y;
    } else v[0] = *p;
}

// Where a wave is: its channels [c0, c0 + 16 CH) of group g up to the group's end, and its lane's places in both mappings.
template <typename T, int CH, int NS, int VE> struct Wave {
    static constexpr int WC = 16 * CH, NP = 4 * NS, PER = TT * WC / 64, NV = PER / VE, NBC = TT * NP / 64;
    int lane, cl, r, g, c0, cend;
    __device__ __forceinline__ Wave(const Args& A, int blk) {
        lane = threadIdx.x;
        cl = lane & 15;
        r = lane >> 4;
        g = blk / A.nblk;
        const int per = A.D / A.G;
        c0 = g * per + (blk % A.nblk) * WC;
        cend = (g + 1) * per;
    }
    __device__ __forceinline__ int channel(int i) const { return c0 + cl * CH + i; }
    // staging: vector k of this lane is token trow(k) of the tile, channels c0 + tcol(k) ...
    __device__ __forceinline__ int trow(int k) const { return (k * 64 + lane) / (WC / VE); }
    __device__ __forceinline__ int tcol(int k) const { return (k * 64 + lane) % (WC / VE) * VE; }
    // (a tile's base is uniform; 8 rows of any tensor span less than 2^31 bytes: the host sees to it)
    __device__ __forceinline__ unsigned place(int k, int row, int t0, int te) const {
        return t0 + trow(k) < te && c0 + tcol(k) < cend ? (trow(k) * row + tcol(k)) * (unsigned)sizeof(T) : BUF_OUT;
    }
    __device__ __forceinline__ bool staged(int k, int v, int t0, int te) const {
        return t0 + trow(k) < te && c0 + tcol(k) + v < cend;
    }
    __device__ __forceinline__ void fetch(const Rows& R, int b, int t0, int te, Raw<T, VE> (&v)[NV]) const {
        const auto rs = buffer_of(static_cast<const T*>(R.p) + b * R.batch + t0 * R.row + c0, BUF_BYTES);
#pragma unroll
        for (int k = 0; k < NV; ++k) v[k] = buf_load<T, VE>(rs, place(k, (int)R.row, t0, te));
    }
    __device__ __forceinline__ void put(void* p, int b, int L, int D, int t0, int te, const Raw<T, VE> (&v)[NV]) const {
        const auto rs = buffer_of(static_cast<T*>(p) + ((long)b * L + t0) * D + c0, BUF_BYTES);
#pragma unroll
        for (int k = 0; k < NV; ++k) buf_store<T, VE>(rs, place(k, D, t0, te), v[k]);
    }
    __device__ __forceinline__ void fetch_bc(const Rows& R, int b, int t0, int te, int N, Raw<T, 1> (&v)[NBC]) const {
        const auto rs = buffer_of(static_cast<const T*>(R.p) + b * R.batch + t0 * R.row + (long)g * N, BUF_BYTES);
#pragma unroll
        for (int k = 0; k < NBC; ++k) {
            const int t = (k * 64 + lane) / NP, n = (k * 64 + lane) % NP;
            v[k] = buf_load<T, 1>(rs, t0 + t < te && n < N ? (t * (int)R.row + n) * (unsigned)sizeof(T) : BUF_OUT);
        }
    }
    // per-channel parameters of the staged channels, in LDS for the whole run
    __device__ __forceinline__ void stage_param(const float* p, float* s) const {
        if (lane < WC) s[lane] = p && c0 + lane < cend ? p[c0 + lane] : 0.f;
    }
    __device__ __forceinline__ void lane_a(const Args& A, float (&a2)[CH][NS]) const {
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                const int n = r * NS + j;
                a2[i][j] = channel(i) < cend && n < A.N ? A.a[(long)channel(i) * A.N + n] * LOG2E : 0.f;
            }
    }
    // a state in its public layout [B][D][N]
    __device__ __forceinline__ void load_state(const float* s, int b, int D, int N, float (&h)[CH][NS]) const {
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                const int n = r * NS + j;
                h[i][j] = s && channel(i) < cend && n < N ? s[((long)b * D + channel(i)) * N + n] : 0.f;
            }
    }
    __device__ __forceinline__ void store_state(float* s, int b, int D, int N, const float (&h)[CH][NS]) const {
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                const int n = r * NS + j;
                if (channel(i) < cend && n < N) s[((long)b * D + channel(i)) * N + n] = h[i][j];
            }
    }
    // ... and in the wave's own: 4 x 16 bytes a lane, lanes side by side
    __device__ __forceinline__ void load_own(const float* p, float (&h)[CH][NS]) const {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const float4 f = *reinterpret_cast<const float4*>(p + (v * 64 + lane) * 4);
            h[v * 4 / NS][v * 4 % NS] = f.x; h[v * 4 / NS][v * 4 % NS + 1] = f.y;
            h[v * 4 / NS][v * 4 % NS + 2] = f.z; h[v * 4 / NS][v * 4 % NS + 3] = f.w;
        }
    }
    __device__ __forceinline__ void store_own(float* p, const float (&h)[CH][NS]) const {
#pragma unroll
        for (int v = 0; v < 4; ++v)
            *reinterpret_cast<float4*>(p + (v * 64 + lane) * 4) =
                make_float4(h[v * 4 / NS][v * 4 % NS], h[v * 4 / NS][v * 4 % NS + 1], h[v * 4 / NS][v * 4 % NS + 2],
                            h[v * 4 / NS][v * 4 % NS + 3]);
    }
};

__device__ __forceinline__ int length_of(const Args& A, int b) {
    return A.lengths ? max(0, min(A.L, A.lengths[b])) : A.L;
}
// dt of staged raw values; 0 past the end (a token that moves no state) and past the channels
template <typename W, typename R, int NV, int VE>
__device__ __forceinline__ void stage_steps(const W& w, const R (&d)[NV], const float* s_bias, int softplus, int t0, int te,
                                            float (&dt)[NV][VE]) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int v = 0; v < VE; ++v) dt[k][v] = d[k].get(v) + s_bias[w.tcol(k) + v];
    if (softplus) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int v = 0; v < VE; ++v) dt[k][v] = softplus_f(dt[k][v]);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int v = 0; v < VE; ++v)
            if (t0 + w.trow(k) >= te || w.c0 + w.tcol(k) + v >= w.cend) dt[k][v] = 0.f;
}
// dy silu(gate)
template <typename W, typename R, int NV, int VE>
__device__ __forceinline__ void stage_core(const R (&gy)[NV], const R (&z)[NV], bool gated, float (&dc)[NV][VE]) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int v = 0; v < VE; ++v) dc[k][v] = gy[k].get(v);
    if (gated) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int v = 0; v < VE; ++v) dc[k][v] *= silu_f(z[k].get(v));
    }
}

// FULL: the forward.  Otherwise the first pass over a segment: its end state from 0, and sum dt.
template <typename T, int CH, int NS, int VE, bool FULL>
__global__ __launch_bounds__(64) void scan_fwd(Args A) {
    typedef Wave<T, CH, NS, VE> W;
    __shared__ __attribute__((aligned(16))) float s_dt[TT * W::WC], s_dtx[TT * W::WC], s_y[FULL ? TT * W::WC : 4],
        s_b[TT * W::NP], s_c[FULL ? TT * W::NP : 4], s_bias[W::WC], s_skip[FULL ? W::WC : 4];
    const int blks = A.nblk * A.G;
    const int blk = blockIdx.x % blks, seg = blockIdx.x / blks % A.segs, b = blockIdx.x / blks / A.segs;
    const W w(A, blk);
    const int len = length_of(A, b), ts = seg * A.seg_len, te = min(A.L, ts + A.seg_len);
    const long wave = ((long)b * blks + blk) * A.segs + seg;
    const int ntile = (A.L + TT - 1) / TT;
    float a2[CH][NS], h[CH][NS], sum_dt[CH];
    w.lane_a(A, a2);
    w.stage_param(A.dt_bias, s_bias);
    if (FULL) w.stage_param(A.skip, s_skip);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        sum_dt[i] = 0.f;
#pragma unroll
        for (int j = 0; j < NS; ++j) h[i][j] = 0.f;
    }
    if (FULL) {
        if (A.segs > 1) w.load_own(A.seg_h + wave * LANE_STATE, h);
        else w.load_state(A.state, b, A.D, A.N, h);
    }
    Raw<T, VE> x[W::NV], d[W::NV], z[W::NV], xn[W::NV], dn[W::NV], zn[W::NV];
    Raw<T, 1> bn[W::NBC], cn[W::NBC];
    auto fetch = [&](int t0) {
        w.fetch(A.x, b, t0, min(len, te), xn);
        w.fetch(A.dt, b, t0, min(len, te), dn);
        w.fetch_bc(A.b, b, t0, min(len, te), A.N, bn);
        if (FULL) {
            if (A.gate.p) w.fetch(A.gate, b, t0, min(len, te), zn);
            w.fetch_bc(A.c, b, t0, min(len, te), A.N, cn);
        }
    };
    fetch(ts);
    for (int t0 = ts; t0 < te; t0 += TT) {
        if (t0 >= len) {                                   // nothing left of this sequence: zero rows
            if (!FULL) break;
#pragma unroll
            for (int k = 0; k < W::NV; ++k) x[k].zero();
            w.put(A.y, b, A.L, A.D, t0, te, x);
            continue;
        }
#pragma unroll
        for (int k = 0; k < W::NV; ++k) { x[k] = xn[k]; d[k] = dn[k]; if (FULL) z[k] = zn[k]; }
        lds_order();                                       // (the last tile's reads are done)
        float step[W::NV][VE];
        stage_steps(w, d, s_bias, A.softplus, t0, min(len, te), step);
#pragma unroll
        for (int k = 0; k < W::NV; ++k)
#pragma unroll
            for (int v = 0; v < VE; ++v) {
                const int at = w.trow(k) * W::WC + w.tcol(k) + v;
                s_dt[at] = step[k][v];
                s_dtx[at] = step[k][v] * x[k].get(v);
            }
#pragma unroll
        for (int k = 0; k < W::NBC; ++k) {
            s_b[k * 64 + w.lane] = bn[k].get(0);
            if (FULL) s_c[k * 64 + w.lane] = cn[k].get(0);
        }
        lds_order();
        if (t0 + TT < te) fetch(t0 + TT);
        if (FULL && A.keep) w.store_own(A.keep + (((long)b * blks + blk) * ntile + t0 / TT) * LANE_STATE, h);
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            float dt[CH], dtx[CH], bv[NS], cv[NS], y[CH];
            lds_read<CH>(s_dt + t * W::WC + w.cl * CH, dt);
            lds_read<CH>(s_dtx + t * W::WC + w.cl * CH, dtx);
            lds_read<NS>(s_b + t * W::NP + w.r * NS, bv);
            if (FULL) lds_read<NS>(s_c + t * W::NP + w.r * NS, cv);
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                y[i] = 0.f;
                if (!FULL) sum_dt[i] += dt[i];
#pragma unroll
                for (int j = 0; j < NS; ++j) {
                    h[i][j] = __builtin_amdgcn_exp2f(dt[i] * a2[i][j]) * h[i][j] + dtx[i] * bv[j];
                    if (FULL) y[i] += h[i][j] * cv[j];
                }
            }
            if (FULL) s_y[t * W::WC + w.cl * CH + own_channel<CH>(w.r)] = sum_states<CH>(y);
        }
        if (FULL) {
            lds_order();
#pragma unroll
            for (int k = 0; k < W::NV; ++k) {
                const int at = w.trow(k) * W::WC + w.tcol(k);
#pragma unroll
                for (int v = 0; v < VE; ++v) {
                    step[k][v] = s_y[at + v] + s_skip[w.tcol(k) + v] * x[k].get(v);
                }
            }
            if (A.gate.p) {
#pragma unroll
                for (int k = 0; k < W::NV; ++k)
#pragma unroll
                    for (int v = 0; v < VE; ++v) step[k][v] *= silu_f(z[k].get(v));
            }
#pragma unroll
            for (int k = 0; k < W::NV; ++k)
#pragma unroll
                for (int v = 0; v < VE; ++v) d[k].set(v, t0 + w.trow(k) < len ? step[k][v] : 0.f);
            w.put(A.y, b, A.L, A.D, t0, te, d);
        }
    }
    if (FULL) {
        if (A.last && seg == A.segs - 1) w.store_state(A.last, b, A.D, A.N, h);
    } else {
        w.store_own(A.seg_h + wave * LANE_STATE, h);
        if (w.r == 0) {
#pragma unroll
            for (int i = 0; i < CH; ++i) A.seg_dt[wave * W::WC + w.cl * CH + i] = sum_dt[i];
        }
    }
}

// Chains the segments: seg_h[s] becomes the state (REV: the adjoint) that comes into segment s.  A wave takes 16 bytes per
// lane of one wave's states; eight segments are in flight.
template <int CH, int NS, bool REV>
__global__ __launch_bounds__(64) void scan_chain(Args A) {
    typedef Wave<float, CH, NS, 1> W;
    const int blks = A.nblk * A.G, v = blockIdx.x & 3, blk = (blockIdx.x >> 2) % blks, b = (blockIdx.x >> 2) / blks;
    const W w(A, blk);
    float a2[CH][NS], h0[CH][NS];
    w.lane_a(A, a2);
    w.load_state(REV ? A.dlast : A.state, b, A.D, A.N, h0);
    float a[4], h[4];
    int chan = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u)                            // (selects with constant indices: v is the same in all lanes)
        if (u == v) {
            chan = u * 4 / NS;
#pragma unroll
            for (int k = 0; k < 4; ++k) { a[k] = a2[u * 4 / NS][u * 4 % NS + k]; h[k] = h0[u * 4 / NS][u * 4 % NS + k]; }
        }
    const long first = ((long)b * blks + blk) * A.segs;
    float4* p = reinterpret_cast<float4*>(A.seg_h + first * LANE_STATE) + v * 64 + w.lane;
    const float* q = A.seg_dt + first * W::WC + w.cl * CH + chan;
    for (int s0 = 0; s0 < A.segs; s0 += 8) {
        float4 e[8];
        float d[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int s = REV ? A.segs - 1 - s0 - u : s0 + u;
            if (s >= 0 && s < A.segs) { e[u] = p[(long)s * (LANE_STATE / 4)]; d[u] = q[(long)s * W::WC]; }
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int s = REV ? A.segs - 1 - s0 - u : s0 + u;
            if (s >= 0 && s < A.segs) {
                p[(long)s * (LANE_STATE / 4)] = make_float4(h[0], h[1], h[2], h[3]);
                h[0] = __builtin_amdgcn_exp2f(d[u] * a[0]) * h[0] + e[u].x;
                h[1] = __builtin_amdgcn_exp2f(d[u] * a[1]) * h[1] + e[u].y;
                h[2] = __builtin_amdgcn_exp2f(d[u] * a[2]) * h[2] + e[u].z;
                h[3] = __builtin_amdgcn_exp2f(d[u] * a[3]) * h[3] + e[u].w;
            }
        }
    }
}

// The backward's first pass over a segment: the adjoint that leaves it at its front when 0 comes in at its end.
template <typename T, int CH, int NS, int VE>
__global__ __launch_bounds__(64) void scan_bwd_ends(Args A) {
    typedef Wave<T, CH, NS, VE> W;
    __shared__ __attribute__((aligned(16))) float s_dt[TT * W::WC], s_g[TT * W::WC], s_c[TT * W::NP],
        s_bias[W::WC];
    const int blks = A.nblk * A.G;
    const int blk = blockIdx.x % blks, seg = blockIdx.x / blks % A.segs, b = blockIdx.x / blks / A.segs;
    const W w(A, blk);
    const int ts = seg * A.seg_len, te = min(length_of(A, b), min(A.L, ts + A.seg_len));
    const long wave = ((long)b * blks + blk) * A.segs + seg;
    float a2[CH][NS], g[CH][NS], sum_dt[CH];
    w.lane_a(A, a2);
    w.stage_param(A.dt_bias, s_bias);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        sum_dt[i] = 0.f;
#pragma unroll
        for (int j = 0; j < NS; ++j) g[i][j] = 0.f;
    }
    Raw<T, VE> dn[W::NV], zn[W::NV], gn[W::NV];
    Raw<T, 1> cn[W::NBC];
    auto fetch = [&](int t0) {
        w.fetch(A.dt, b, t0, te, dn);
        if (A.gate.p) w.fetch(A.gate, b, t0, te, zn);
        w.fetch(A.dy, b, t0, te, gn);
        w.fetch_bc(A.c, b, t0, te, A.N, cn);
    };
    int t0 = ts + (te - ts - 1) / TT * TT;
    if (te > ts) fetch(t0);
    for (; te > ts && t0 >= ts; t0 -= TT) {
        lds_order();
        float step[W::NV][VE], dcore[W::NV][VE];
        stage_steps(w, dn, s_bias, A.softplus, t0, te, step);
        stage_core<W>(gn, zn, A.gate.p != nullptr, dcore);
#pragma unroll
        for (int k = 0; k < W::NV; ++k)
#pragma unroll
            for (int v = 0; v < VE; ++v) {
                s_dt[w.trow(k) * W::WC + w.tcol(k) + v] = step[k][v];
                s_g[w.trow(k) * W::WC + w.tcol(k) + v] = dcore[k][v];
            }
#pragma unroll
        for (int k = 0; k < W::NBC; ++k) s_c[k * 64 + w.lane] = cn[k].get(0);
        lds_order();
        if (t0 > ts) fetch(t0 - TT);
#pragma unroll
        for (int t = TT - 1; t >= 0; --t) {
            float dt[CH], dc[CH], cv[NS];
            lds_read<CH>(s_dt + t * W::WC + w.cl * CH, dt);
            lds_read<CH>(s_g + t * W::WC + w.cl * CH, dc);
            lds_read<NS>(s_c + t * W::NP + w.r * NS, cv);
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                sum_dt[i] += dt[i];
#pragma unroll
                for (int j = 0; j < NS; ++j)
                    g[i][j] = __builtin_amdgcn_exp2f(dt[i] * a2[i][j]) * (g[i][j] + dc[i] * cv[j]);
            }
        }
    }
    w.store_own(A.seg_h + wave * LANE_STATE, g);
    if (w.r == 0) {
#pragma unroll
        for (int i = 0; i < CH; ++i) A.seg_dt[wave * W::WC + w.cl * CH + i] = sum_dt[i];
    }
}

// The backward.  Tiles from the last to the first; inside a tile the states are computed again from the kept one, forwards,
// staying in registers (h before each of the TT tokens), then the adjoint runs backwards over them.
// One wave takes the sequences of its batch group one after the other, so that its sums over tokens leave once:
// part_p[(group * segs + seg)][block]{da: LANE_STATE, dskip: WC, ddt_bias: WC}; part_bc[block of group][B][L][G][2][N].
template <typename T, int CH, int NS, int VE>
__global__ __launch_bounds__(64, 2) void scan_bwd(Args A) {
    typedef Wave<T, CH, NS, VE> W;
    // s_dtx's row of a token is read for the last time where s_gb's is written, so they share their place
    __shared__ __attribute__((aligned(16))) float s_dt[TT * W::WC], s_dtx[TT * W::WC], s_g[TT * W::WC], s_y[TT * W::WC],
        s_ta[TT * W::WC], s_b[TT * W::NP], s_c[TT * W::NP], s_db[TT * W::NP], s_dc[TT * W::NP], s_bias[W::WC],
        s_skip[W::WC], s_sum[2][W::PER * 64];
    float* s_gb = s_dtx;
    const int blks = A.nblk * A.G;
    const int blk = blockIdx.x % blks, seg = blockIdx.x / blks % A.segs, group = blockIdx.x / blks / A.segs;
    const W w(A, blk);
    const int ntile = (A.L + TT - 1) / TT, ts = seg * A.seg_len, tend = min(A.L, ts + A.seg_len);
    float a2[CH][NS], g[CH][NS], da[CH][NS];
    w.lane_a(A, a2);
    w.stage_param(A.dt_bias, s_bias);
    w.stage_param(A.skip, s_skip);
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int j = 0; j < NS; ++j) da[i][j] = 0.f;
#pragma unroll
    for (int k = 0; k < W::PER; ++k) s_sum[0][k * 64 + w.lane] = s_sum[1][k * 64 + w.lane] = 0.f;
    lds_order();
    for (int b = group; b < A.B; b += A.bgroups) {
        const int len = length_of(A, b), te = min(len, tend);
        if (A.segs > 1) w.load_own(A.seg_h + (((long)b * blks + blk) * A.segs + seg) * LANE_STATE, g);
        else w.load_state(A.dlast, b, A.D, A.N, g);
        for (int t0 = ts + (tend - ts - 1) / TT * TT; t0 >= ts; t0 -= TT) {
            Raw<T, VE> x[W::NV], d[W::NV], z[W::NV], gy[W::NV];
            if (t0 >= te) {                                // past the end of this sequence: zero rows
#pragma unroll
                for (int k = 0; k < W::NV; ++k) x[k].zero();
                w.put(A.dx, b, A.L, A.D, t0, tend, x);
                w.put(A.ddt, b, A.L, A.D, t0, tend, x);
                if (A.gate.p) w.put(A.dgate, b, A.L, A.D, t0, tend, x);
                continue;
            }
            float hist[TT][CH][NS], h[CH][NS];
            w.load_own(A.keep + (((long)b * blks + blk) * ntile + t0 / TT) * LANE_STATE, h);
            w.fetch(A.x, b, t0, te, x);
            w.fetch(A.dt, b, t0, te, d);
            if (A.gate.p) w.fetch(A.gate, b, t0, te, z);
            w.fetch(A.dy, b, t0, te, gy);
            Raw<T, 1> br[W::NBC], cr[W::NBC];
            w.fetch_bc(A.b, b, t0, te, A.N, br);
            w.fetch_bc(A.c, b, t0, te, A.N, cr);
            lds_order();
            {
                float step[W::NV][VE], dcore[W::NV][VE];
                stage_steps(w, d, s_bias, A.softplus, t0, te, step);
                stage_core<W>(gy, z, A.gate.p != nullptr, dcore);
#pragma unroll
                for (int k = 0; k < W::NV; ++k)
#pragma unroll
                    for (int v = 0; v < VE; ++v) {
                        const int at = w.trow(k) * W::WC + w.tcol(k) + v;
                        s_dt[at] = step[k][v];
                        s_dtx[at] = step[k][v] * x[k].get(v);
                        s_g[at] = dcore[k][v];
                    }
            }
#pragma unroll
            for (int k = 0; k < W::NBC; ++k) {
                s_b[k * 64 + w.lane] = br[k].get(0);
                s_c[k * 64 + w.lane] = cr[k].get(0);
            }
            lds_order();
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                float dt[CH], dtx[CH], dc[CH], bv[NS], cv[NS], y[CH], sc[NS];
                lds_read<CH>(s_dt + t * W::WC + w.cl * CH, dt);
                lds_read<CH>(s_dtx + t * W::WC + w.cl * CH, dtx);
                lds_read<CH>(s_g + t * W::WC + w.cl * CH, dc);
                lds_read<NS>(s_b + t * W::NP + w.r * NS, bv);
                lds_read<NS>(s_c + t * W::NP + w.r * NS, cv);
#pragma unroll
                for (int j = 0; j < NS; ++j) sc[j] = 0.f;
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    y[i] = 0.f;
#pragma unroll
                    for (int j = 0; j < NS; ++j) {
                        hist[t][i][j] = h[i][j];
                        h[i][j] = __builtin_amdgcn_exp2f(dt[i] * a2[i][j]) * h[i][j] + dtx[i] * bv[j];
                        y[i] += h[i][j] * cv[j];
                        sc[j] += h[i][j] * dc[i];
                    }
                }
                s_y[t * W::WC + w.cl * CH + own_channel<CH>(w.r)] = sum_states<CH>(y);
#pragma unroll
                for (int j = 0; j < NS; j += 4) sum16_x4(sc[j], sc[j + 1], sc[j + 2], sc[j + 3]);
                if (w.cl == 0) {
#pragma unroll
                    for (int j = 0; j < NS; ++j) s_dc[t * W::NP + w.r * NS + j] = sc[j];
                }
                __builtin_amdgcn_sched_barrier(0);         // (later tokens' LDS reads would take registers hist needs)
            }
            lds_order();                                   // (and the decays are formed again, not held in 128 registers)
#pragma unroll
            for (int t = TT - 1; t >= 0; --t) {
                if (t == TT / 2 - 1) {                     // (the rows again, from L2: half of hist's registers are free now)
                    w.fetch(A.x, b, t0, te, x);
                    w.fetch(A.dt, b, t0, te, d);
                    if (A.gate.p) w.fetch(A.gate, b, t0, te, z);
                    w.fetch(A.dy, b, t0, te, gy);
                }
                float dt[CH], dtx[CH], dc[CH], bv[NS], cv[NS], gb[CH], ta[CH], sb[NS];
                lds_read<CH>(s_dt + t * W::WC + w.cl * CH, dt);
                lds_read<CH>(s_dtx + t * W::WC + w.cl * CH, dtx);
                lds_read<CH>(s_g + t * W::WC + w.cl * CH, dc);
                lds_read<NS>(s_b + t * W::NP + w.r * NS, bv);
                lds_read<NS>(s_c + t * W::NP + w.r * NS, cv);
#pragma unroll
                for (int j = 0; j < NS; ++j) sb[j] = 0.f;
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    gb[i] = ta[i] = 0.f;
#pragma unroll
                    for (int j = 0; j < NS; ++j) {
                        const float G = g[i][j] + dc[i] * cv[j];
                        gb[i] += G * bv[j];
                        sb[j] += G * dtx[i];
                        g[i][j] = G * __builtin_amdgcn_exp2f(dt[i] * a2[i][j]);
                        const float th = g[i][j] * hist[t][i][j];
                        ta[i] += th * a2[i][j];
                        da[i][j] += th * dt[i];
                    }
                }
                s_gb[t * W::WC + w.cl * CH + own_channel<CH>(w.r)] = sum_states<CH>(gb);
                s_ta[t * W::WC + w.cl * CH + own_channel<CH>(w.r)] = sum_states<CH>(ta);
#pragma unroll
                for (int j = 0; j < NS; j += 4) sum16_x4(sb[j], sb[j + 1], sb[j + 2], sb[j + 3]);
                if (w.cl == 0) {
#pragma unroll
                    for (int j = 0; j < NS; ++j) s_db[t * W::NP + w.r * NS + j] = sb[j];
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            lds_order();
#pragma unroll
            for (int k = 0; k < W::NBC; ++k) {
                const int t = (k * 64 + w.lane) / W::NP, n = (k * 64 + w.lane) % W::NP;
                const auto rs = buffer_of(
                    A.part_bc + ((((long)(blk % A.nblk) * A.B + b) * A.L + t0) * A.G + w.g) * 2 * A.N, BUF_BYTES);
                const unsigned at = t0 + t < te && n < A.N ? (t * A.G * 2 * A.N + n) * 4u : BUF_OUT;
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(s_db[k * 64 + w.lane]), rs, at, 0, 0);
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(s_dc[k * 64 + w.lane]), rs, at, A.N * 4, 0);
            }
            float dr[W::NV][VE], core[W::NV][VE];
#pragma unroll
            for (int k = 0; k < W::NV; ++k)
#pragma unroll
                for (int v = 0; v < VE; ++v) {
                    const int at = w.trow(k) * W::WC + w.tcol(k) + v;
                    dr[k][v] = s_ta[at] * LN2 + x[k].get(v) * s_gb[at];
                    core[k][v] = s_y[at] + s_skip[w.tcol(k) + v] * x[k].get(v);
                }
            if (A.softplus) {                              // softplus' = sigmoid, from the side that does not overflow
#pragma unroll
                for (int k = 0; k < W::NV; ++k)
#pragma unroll
                    for (int v = 0; v < VE; ++v) {
                        const float u = d[k].get(v) + s_bias[w.tcol(k) + v], e = exp_f(-fabsf(u));
                        dr[k][v] *= (u < 0.f ? e : 1.f) * __builtin_amdgcn_rcpf(1.f + e);
                    }
            }
            if (A.gate.p) {
#pragma unroll
                for (int k = 0; k < W::NV; ++k)
#pragma unroll
                    for (int v = 0; v < VE; ++v)
                        z[k].set(v, w.staged(k, v, t0, te) ? gy[k].get(v) * core[k][v] * dsilu_f(z[k].get(v)) : 0.f);
                w.put(A.dgate, b, A.L, A.D, t0, tend, z);
            }
#pragma unroll
            for (int k = 0; k < W::NV; ++k)
#pragma unroll
                for (int v = 0; v < VE; ++v) {
                    const int at = w.trow(k) * W::WC + w.tcol(k) + v;
                    const bool on = w.staged(k, v, t0, te);
                    const float dc = s_g[at], e = on ? dr[k][v] : 0.f;
                    s_sum[0][(k * 64 + w.lane) * VE + v] += on ? dc * x[k].get(v) : 0.f;
                    s_sum[1][(k * 64 + w.lane) * VE + v] += e;
                    x[k].set(v, on ? s_dt[at] * s_gb[at] + s_skip[w.tcol(k) + v] * dc : 0.f);
                    d[k].set(v, e);
                }
            w.put(A.dx, b, A.L, A.D, t0, tend, x);
            w.put(A.ddt, b, A.L, A.D, t0, tend, d);
        }
        if (A.dstate && seg == 0) w.store_state(A.dstate, b, A.D, A.N, g);
    }
    float* out = A.part_p + (((long)group * A.segs + seg) * blks + blk) * (LANE_STATE + 2 * W::WC);
    w.store_own(out, da);
    // sums over the tokens of a tile: lanes that staged the same channels meet in LDS
    for (int half = 0; half < 2; ++half) {
        lds_order();
#pragma unroll
        for (int k = 0; k < W::NV; ++k)
#pragma unroll
            for (int v = 0; v < VE; ++v)
                s_dt[w.trow(k) * W::WC + w.tcol(k) + v] = s_sum[half][(k * 64 + w.lane) * VE + v];
        lds_order();
        if (w.lane < W::WC) {
            float s = 0.f;
#pragma unroll
            for (int t = 0; t < TT; ++t) s += s_dt[t * W::WC + w.lane];
            out[LANE_STATE + half * W::WC + w.lane] = s;
        }
    }
}

// part_p's rows summed in a fixed order (16 row lanes x 64 columns) and put in their public places.
template <int CH, int NS>
__global__ __launch_bounds__(1024) void scan_params(const float* __restrict__ part, int rows, int D, int N, int G,
                                                    int nblk, float* __restrict__ da, float* __restrict__ dskip,
                                                    float* __restrict__ dbias) {
    constexpr int WC = 16 * CH, PER = LANE_STATE + 2 * WC;
    const long cols = (long)nblk * G * PER, col = (long)blockIdx.x * 64 + (threadIdx.x & 63);
    const int lr = threadIdx.x >> 6;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    if (col < cols)
        for (int r = lr; r < rows; r += 64) {
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (r + 16 * u < rows) acc[u] += part[(r + 16 * u) * cols + col];
        }
    __shared__ float s[16][64];
    s[lr][threadIdx.x & 63] = (acc[0] + acc[1]) + (acc[2] + acc[3]);
    __syncthreads();
    if (lr != 0 || col >= cols) return;
    float t = 0.f;
#pragma unroll
    for (int u = 0; u < 16; ++u) t += s[u][threadIdx.x];
    const int blk = (int)(col / PER), e = (int)(col % PER), per = D / G, g = blk / nblk;
    const int c0 = g * per + blk % nblk * WC, cend = (g + 1) * per;
    if (e < LANE_STATE) {
        const int v = e / 256, lane = e / 4 % 64, k = v * 4 + e % 4;       // element k of the lane's CH x NS states
        const int c = c0 + (lane & 15) * CH + k / NS, n = (lane >> 4) * NS + k % NS;
        if (c < cend && n < N) da[(long)c * N + n] = t;
    } else {
        const int q = e - LANE_STATE, c = c0 + q % WC;
        if (c < cend) {
            if (q < WC) { if (dskip) dskip[c] = t; }
            else if (dbias) dbias[c] = t;
        }
    }
}

// db and dc: the channel blocks' shares in a fixed order; rows past a sequence's length are 0
template <typename T>
__global__ __launch_bounds__(256) void scan_shared(const float* __restrict__ part, const int* __restrict__ lengths, int B,
                                                   int L, int G, int N, int nblk, T* __restrict__ db, T* __restrict__ dc) {
    const long n = (long)B * L * G * 2 * N, id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= n) return;
    const long tok = id / (2 * N * G);
    float s = 0.f;
    if (!lengths || (int)(tok % L) < lengths[tok / L])
        for (int k = 0; k < nblk; ++k) s += part[k * n + id];
    const long row = id / (2 * N);
    const int e = (int)(id % (2 * N));
    (e < N ? db[row * N + e] : dc[row * N + e - N]) = from_f32<T>(s);
}

// One token: a lane takes four states of a channel, LN lanes a channel.  Bound by the state's bytes, read and written once.
template <typename T, int LN, bool VEC>
__global__ __launch_bounds__(256) void scan_token(Rows x, float* __restrict__ state, long state_batch, Rows dt, Rows gate,
                                                  Rows b, Rows c, const float* __restrict__ a,
                                                  const float* __restrict__ skip, const float* __restrict__ dt_bias,
                                                  int softplus, int B, int D, int N, int G, T* __restrict__ y) {
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    const int part = (int)(id % LN);
    const long ch = id / LN;
    if (ch >= (long)B * D) return;                         // (whole channels: the LN lanes stay together)
    const int d = (int)(ch % D), bi = (int)(ch / D), g = d / (D / G), n0 = part * 4;
    const T* bp = static_cast<const T*>(b.p) + bi * b.batch + (long)g * N;
    const T* cp = static_cast<const T*>(c.p) + bi * c.batch + (long)g * N;
    float* hp = state + bi * state_batch + (long)d * N;
    float h[4], av[4], bv[4], cv[4];
    if constexpr (VEC) {
        if (n0 < N) {
            const float4 t = *reinterpret_cast<const float4*>(hp + n0), u = *reinterpret_cast<const float4*>(a + (long)d * N + n0);
            h[0] = t.x; h[1] = t.y; h[2] = t.z; h[3] = t.w;
            av[0] = u.x; av[1] = u.y; av[2] = u.z; av[3] = u.w;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) h[k] = av[k] = 0.f;
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            h[k] = n0 + k < N ? hp[n0 + k] : 0.f;
            av[k] = n0 + k < N ? a[(long)d * N + n0 + k] : 0.f;
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        bv[k] = n0 + k < N ? to_f32(bp[n0 + k]) : 0.f;
        cv[k] = n0 + k < N ? to_f32(cp[n0 + k]) : 0.f;
    }
    const float xv = to_f32(static_cast<const T*>(x.p)[bi * x.batch + d]);
    float step = to_f32(static_cast<const T*>(dt.p)[bi * dt.batch + d]) + (dt_bias ? dt_bias[d] : 0.f);
    if (softplus) step = softplus_f(step);
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        h[k] = exp_f(step * av[k]) * h[k] + step * xv * bv[k];
        s += h[k] * cv[k];
    }
    if constexpr (VEC) {
        if (n0 < N) *reinterpret_cast<float4*>(hp + n0) = make_float4(h[0], h[1], h[2], h[3]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (n0 + k < N) hp[n0 + k] = h[k];
    }
#pragma unroll
    for (int o = 1; o < LN; o <<= 1) s += __shfl_xor(s, o);
    if (part == 0) {
        if (skip) s += skip[d] * xv;
        if (gate.p) s *= silu_f(to_f32(static_cast<const T*>(gate.p)[bi * gate.batch + d]));
        y[(long)bi * D + d] = from_f32<T>(s);
    }
}

// Channels a lane holds: CH x NS = 16 values, NS states a lane over 4 rows.
int ch_of(int N) { return N <= 16 ? 4 : N <= 32 ? 2 : 1; }
int blocks_of(int D, int G, int N) { return (D / G + 16 * ch_of(N) - 1) / (16 * ch_of(N)); }

// Segments: none while the waves of whole sequences keep the chip's 1024 SIMDs busy; else enough for some 4096 waves, each
// of 8 tiles at least.
void cut(int B, int L, int D, int G, int N, int& segs, int& seg_len) {
    const long waves = (long)B * G * blocks_of(D, G, N);
    long s = waves >= 1024 ? 1 : 4096 / waves;
    const long most = L / (8 * TT);
    if (s > most) s = most;
    if (s < 1) s = 1;
    long len = (L + s - 1) / s;
    len = (len + TT - 1) / TT * TT;
    seg_len = (int)len;
    segs = (int)((L + len - 1) / len);
}
int batch_groups(int B, int L, int D, int G, int N) {
    int segs, len;
    cut(B, L, D, G, N, segs, len);
    const long waves = (long)G * blocks_of(D, G, N) * segs;
    const long g = 4096 / waves;
    return (int)(g < 1 ? 1 : g > B ? B : g);
}

bool bad_shape(int dtype, int B, int L, int D, int N, int G) {
    return !vqa_dtype_ok(dtype) || B < 1 || L < 1 || L > 0x3fffffff || D < 1 || N < 1 || N > 64 || G < 1 || D % G != 0 ||
           (double)B * L > 1e9 || (double)B * L * D > 4e11 || (double)B * D > 1e10 || (double)B * L * G * N > 1e11 ||
           (double)G * blocks_of(D, G, N) * B > 2e8;
}
// (buffer accesses of up to 16 bytes want their addresses on 4 bytes)
bool on4(const void* p, long stride, int e) { return ((uintptr_t)p & 3) == 0 && stride * e % 4 == 0; }
bool rows_vec(const Rows& r, int e) { return !r.p || (on4(r.p, r.batch, e) && on4(r.p, r.row, e)); }
bool far_rows(const Rows& r) { return r.p && (r.row < 0 || r.row > 0x7fffffffL / (4 * TT)); }
bool far_rows(const Args& A) {
    return far_rows(A.x) || far_rows(A.dt) || far_rows(A.gate) || far_rows(A.b) || far_rows(A.c) || far_rows(A.dy) ||
           A.D > 0x7fffffff / (4 * TT) || (long)A.G * A.N > 0x7fffffff / (8 * TT);
}
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <typename T, int CH, int NS, int VE> int launch(int kind, const Args& A, hipStream_t st) {
    const long blks = (long)A.nblk * A.G;
    if (kind == 0) {
        if (A.segs > 1) {
            scan_fwd<T, CH, NS, VE, false><<<(unsigned)(blks * A.segs * A.B), 64, 0, st>>>(A);
            CHECK_LAUNCH();
            scan_chain<CH, NS, false><<<(unsigned)(blks * A.B * 4), 64, 0, st>>>(A);
            CHECK_LAUNCH();
        }
        scan_fwd<T, CH, NS, VE, true><<<(unsigned)(blks * A.segs * A.B), 64, 0, st>>>(A);
    } else {
        if (A.segs > 1) {
            scan_bwd_ends<T, CH, NS, VE><<<(unsigned)(blks * A.segs * A.B), 64, 0, st>>>(A);
            CHECK_LAUNCH();
            scan_chain<CH, NS, true><<<(unsigned)(blks * A.B * 4), 64, 0, st>>>(A);
            CHECK_LAUNCH();
        }
        scan_bwd<T, CH, NS, VE><<<(unsigned)(blks * A.segs * A.bgroups), 64, 0, st>>>(A);
    }
    CHECK_LAUNCH();
    return VQA_OK;
}
template <typename T> int by_states(int kind, bool vec, const Args& A, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    if (A.N <= 16) return vec ? launch<T, 4, 4, V>(kind, A, st) : launch<T, 4, 4, 1>(kind, A, st);
    if (A.N <= 32) return vec ? launch<T, 2, 8, 4>(kind, A, st) : launch<T, 2, 8, 1>(kind, A, st);
    return vec ? launch<T, 1, 16, 2>(kind, A, st) : launch<T, 1, 16, 1>(kind, A, st);
}
int by_type(int kind, int dtype, bool vec, const Args& A, hipStream_t st) {
    if (dtype == VQA_F32) return by_states<float>(kind, vec, A, st);
    if (dtype == VQA_BF16) return by_states<bf16>(kind, vec, A, st);
    return by_states<_Float16>(kind, vec, A, st);
}

void plan(Args& A) {
    A.nblk = blocks_of(A.D, A.G, A.N);
    cut(A.B, A.L, A.D, A.G, A.N, A.segs, A.seg_len);
    A.bgroups = batch_groups(A.B, A.L, A.D, A.G, A.N);
}
// Workspace, in floats: the segments' states and sums of dt (none without segments), the backward's partial sums
long seg_floats(const Args& A) {
    return A.segs > 1 ? (long)A.B * A.nblk * A.G * A.segs * (LANE_STATE + 16 * ch_of(A.N)) : 0;
}
long part_p_floats(const Args& A) {
    return (long)A.bgroups * A.segs * A.nblk * A.G * (LANE_STATE + 32 * ch_of(A.N));
}
long part_bc_floats(const Args& A) { return (long)A.nblk * A.B * A.L * A.G * 2 * A.N; }

}  // namespace

extern "C" int vqa_scan_ws_bytes(int dtype, int B, int L, int D, int N, int G, long* sizes) {
    if (bad_shape(dtype, B, L, D, N, G) || !sizes) return VQA_ERR_ARG;
    Args A = {};
    A.B = B; A.L = L; A.D = D; A.N = N; A.G = G;
    plan(A);
    sizes[0] = 4 * seg_floats(A);
    sizes[1] = 4L * B * A.nblk * G * ((L + TT - 1) / TT) * LANE_STATE;
    sizes[2] = 4 * (seg_floats(A) + part_p_floats(A) + part_bc_floats(A));
    return VQA_OK;
}

extern "C" int vqa_scan_fwd(void* stream, int dtype, const void* x, long x_batch, long x_row, const void* dt,
                            long dt_batch, long dt_row, const void* gate, long gate_batch, long gate_row, const float* a,
                            const void* b, long b_batch, long b_row, const void* c, long c_batch, long c_row,
                            const float* skip, const float* dt_bias, int softplus, const float* state,
                            const int* lengths, int B, int L, int D, int N, int G, void* y, float* last, float* keep,
                            float* ws) {
    if (bad_shape(dtype, B, L, D, N, G) || !x || !dt || !a || !b || !c || !y) return VQA_ERR_ARG;
    Args A = {};
    A.x = {x, x_batch, x_row}; A.dt = {dt, dt_batch, dt_row}; A.gate = {gate, gate_batch, gate_row};
    A.b = {b, b_batch, b_row}; A.c = {c, c_batch, c_row};
    A.a = a; A.skip = skip; A.dt_bias = dt_bias; A.state = state; A.lengths = lengths; A.softplus = softplus;
    A.B = B; A.L = L; A.D = D; A.N = N; A.G = G; A.y = y; A.last = last; A.keep = keep;
    plan(A);
    if ((A.segs > 1 && !ws) || !aligned16(ws) || !aligned16(keep) || far_rows(A)) return VQA_ERR_ARG;
    A.seg_h = ws;
    A.seg_dt = ws ? ws + (long)B * A.nblk * G * A.segs * LANE_STATE : nullptr;
    const int e = vqa_elem_bytes(dtype);
    const bool vec = (D / G) % (16 / e) == 0 && rows_vec(A.x, e) && rows_vec(A.dt, e) && rows_vec(A.gate, e) &&
                     on4(y, D, e);
    return by_type(0, dtype, vec, A, static_cast<hipStream_t>(stream));
}

extern "C" int vqa_scan_bwd(void* stream, int dtype, const void* dy, long dy_batch, long dy_row, const float* dlast,
                            const void* x, long x_batch, long x_row, const void* dt, long dt_batch, long dt_row,
                            const void* gate, long gate_batch, long gate_row, const float* a, const void* b, long b_batch,
                            long b_row, const void* c, long c_batch, long c_row, const float* skip, const float* dt_bias,
                            int softplus, const int* lengths, int B, int L, int D, int N, int G, const float* keep,
                            void* dx, void* ddt, void* dgate, float* da, void* db, void* dc, float* dskip,
                            float* ddt_bias, float* dstate, float* ws) {
    if (bad_shape(dtype, B, L, D, N, G) || !dy || !x || !dt || !a || !b || !c || !keep || !dx || !ddt || !da || !db ||
        !dc || !ws || (gate && !dgate) || !aligned16(ws) || !aligned16(keep))
        return VQA_ERR_ARG;
    Args A = {};
    A.dy = {dy, dy_batch, dy_row};
    A.x = {x, x_batch, x_row}; A.dt = {dt, dt_batch, dt_row}; A.gate = {gate, gate_batch, gate_row};
    A.b = {b, b_batch, b_row}; A.c = {c, c_batch, c_row};
    A.a = a; A.skip = skip; A.dt_bias = dt_bias; A.dlast = dlast; A.lengths = lengths; A.softplus = softplus;
    A.B = B; A.L = L; A.D = D; A.N = N; A.G = G; A.keep = const_cast<float*>(keep);
    A.dx = dx; A.ddt = ddt; A.dgate = dgate; A.dstate = dstate;
    if (far_rows(A)) return VQA_ERR_ARG;
    plan(A);
    A.seg_h = ws;
    A.seg_dt = ws + (A.segs > 1 ? (long)B * A.nblk * G * A.segs * LANE_STATE : 0);
    A.part_p = ws + seg_floats(A);
    A.part_bc = A.part_p + part_p_floats(A);
    const int e = vqa_elem_bytes(dtype);
    const bool vec = (D / G) % (16 / e) == 0 && rows_vec(A.x, e) && rows_vec(A.dt, e) && rows_vec(A.gate, e) &&
                     rows_vec(A.dy, e) && on4(dx, D, e) && on4(ddt, D, e) && on4(dgate, D, e);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const int rc = by_type(1, dtype, vec, A, st);
    if (rc != VQA_OK) return rc;
    const int rows = A.bgroups * A.segs;
    const long cols = (long)A.nblk * G * (LANE_STATE + 32 * ch_of(N));
    const unsigned pg = (unsigned)((cols + 63) / 64);
    if (N <= 16) scan_params<4, 4><<<pg, 1024, 0, st>>>(A.part_p, rows, D, N, G, A.nblk, da, dskip, ddt_bias);
    else if (N <= 32) scan_params<2, 8><<<pg, 1024, 0, st>>>(A.part_p, rows, D, N, G, A.nblk, da, dskip, ddt_bias);
    else scan_params<1, 16><<<pg, 1024, 0, st>>>(A.part_p, rows, D, N, G, A.nblk, da, dskip, ddt_bias);
    CHECK_LAUNCH();
    const unsigned sg = (unsigned)(((long)B * L * G * 2 * N + 255) / 256);
    if (dtype == VQA_F32) scan_shared<float><<<sg, 256, 0, st>>>(A.part_bc, lengths, B, L, G, N, A.nblk, static_cast<float*>(db), static_cast<float*>(dc));
    else if (dtype == VQA_BF16) scan_shared<bf16><<<sg, 256, 0, st>>>(A.part_bc, lengths, B, L, G, N, A.nblk, static_cast<bf16*>(db), static_cast<bf16*>(dc));
    else scan_shared<_Float16><<<sg, 256, 0, st>>>(A.part_bc, lengths, B, L, G, N, A.nblk, static_cast<_Float16*>(db), static_cast<_Float16*>(dc));
    CHECK_LAUNCH();
    return VQA_OK;
}

namespace {
template <typename T>
int token(hipStream_t st, const Rows& x, float* state, long sb, const Rows& dt, const Rows& gate, const Rows& b, const Rows& c,
          const float* a, const float* skip, const float* bias, int softplus, int B, int D, int N, int G, void* y) {
    const bool vec = N % 4 == 0 && sb % 4 == 0 && aligned16(state) && aligned16(a);
    const int ln = N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16;
    const unsigned grid = (unsigned)(((long)B * D * ln + 255) / 256);
#define VQA_TOKEN(LN)                                                                                                    \
    if (ln == LN) {                                                                                                      \
        if (vec) scan_token<T, LN, true><<<grid, 256, 0, st>>>(x, state, sb, dt, gate, b, c, a, skip, bias, softplus, B, D, N, G, static_cast<T*>(y)); \
        else scan_token<T, LN, false><<<grid, 256, 0, st>>>(x, state, sb, dt, gate, b, c, a, skip, bias, softplus, B, D, N, G, static_cast<T*>(y));    \
    }
    VQA_TOKEN(1) VQA_TOKEN(2) VQA_TOKEN(4) VQA_TOKEN(8) VQA_TOKEN(16)
#undef VQA_TOKEN
    CHECK_LAUNCH();
    return VQA_OK;
}
}  // namespace

extern "C" int vqa_scan_token(void* stream, int dtype, const void* x, long x_batch, float* state, long state_batch,
                              const void* dt, long dt_batch, const void* gate, long gate_batch, const float* a,
                              const void* b, long b_batch, const void* c, long c_batch, const float* skip,
                              const float* dt_bias, int softplus, int B, int D, int N, int G, void* y) {
    if (bad_shape(dtype, B, 1, D, N, G) || !x || !state || !dt || !a || !b || !c || !y) return VQA_ERR_ARG;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const Rows rx = {x, x_batch, 0}, rd = {dt, dt_batch, 0}, rg = {gate, gate_batch, 0}, rb = {b, b_batch, 0}, rc = {c, c_batch, 0};
    if (dtype == VQA_F32) return token<float>(st, rx, state, state_batch, rd, rg, rb, rc, a, skip, dt_bias, softplus, B, D, N, G, y);
    if (dtype == VQA_BF16) return token<bf16>(st, rx, state, state_batch, rd, rg, rb, rc, a, skip, dt_bias, softplus, B, D, N, G, y);
    return token<_Float16>(st, rx, state, state_batch, rd, rg, rb, rc, a, skip, dt_bias, softplus, B, D, N, G, y);
}
