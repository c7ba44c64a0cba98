// The selective state space scan: forward, backward and for one token.  Per channel d with states n < N (N <= 64):
//   dt_t = softplus(raw_t + dt_bias);  h_t[n] = exp(dt_t a[n]) h_{t-1}[n] + (dt_t x_t) b_t[n]
//   core_t = sum_n c_t[n] h_t[n] + skip x_t;  y_t = core_t silu(gate_t)
// b and c are shared by the channels of a group.  With dcore = dy silu(gate), G_t the gradient of h_t:
//   G_t = dcore_t c_t + exp(dt_{t+1} a) G_{t+1};  th_t = G_t exp(dt_t a) h_{t-1}
//   dx = dt sum_n G b + skip dcore;  draw = (sum_n a th + x sum_n G b) softplus'(raw + dt_bias);  da = sum_t dt th
//   db_t = sum_d G dt x;  dc_t = sum_d h dcore;  dgate = dy core silu'(gate);  dskip = sum dcore x;  ddt_bias = sum draw
// Tokens at or past a sequence's length: dt = 0 (the state stands still), rows and gradients 0; what lies there is never read
// into a sum (left out by the load, not multiplied by 0).
//
// Arithmetic, not memory, bounds it: N exponentials (two issue slots each) and 4 N other operations per (token, channel)
// against 8 bytes.  It stays in f32 on the vector ALU (the decay differs per channel AND state, so there is no matrix
// product in it).  One wave works on 16 CH channels: lane = 16 channel lanes x 4 state rows, each lane holding CH channels
// x NS states in registers.  What a token needs per channel (dt, dt x, ...) and per state (b, c) is staged in LDS in f32, TT
// tokens at a time, by a second mapping of the lanes in which global rows are read up to 16 bytes a lane; the next tile's
// rows are in flight meanwhile.  Sums over states are lane swaps, sums over channels DPP adds.
// With few rows the tokens are cut into segments: a first pass finds each segment's own end state and total decay (the
// product of decays is exp(a sum dt)), a small one chains them, and the full pass starts every segment from its true
// state.  The backward does the same from the other end.  For the backward the forward keeps h before every tile but the first.
// States in workspaces lie as [..][channel, per_pad of them a group][NP], NP = 8, 16, 32 or 64 >= N.
#include <algorithm>
#include "seq.h"

namespace {

typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));
constexpr int TT = 8;                      // tokens of a tile
constexpr int BW = 4;                      // waves of a backward workgroup
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

enum { SOFTPLUS = 1, SKIP = 2 };
struct Rows { const void* p; long batch, row; };          // [B][L][...], element strides; the last axis is contiguous

struct Args {
    Rows x, dt, gate, b, c, dy;
    const float *a, *skip, *dt_bias, *state, *dlast;
    const int* lengths;
    int flags, B, L, D, N, G;              // flags: SOFTPLUS, SKIP (there is one)
    int per, per_pad, fblk, bblk;          // channels of a group, padded; forward waves, backward workgroups across it
    int segs, seg_len, bgroups;            // segments, tokens of one, batch groups of the backward
    bool narrow;                           // forward waves of half the channels
    void* y; float* last;
    float *keep, *seg_h, *seg_dt;          // h before the tiles; per segment: state, then the true incoming one; sum dt
    void *dx, *ddt, *dgate; float *part_bc, *part_p, *dstate;
    void *db, *dc; float *da, *dskip, *dbias; int params;      // the join's outputs, its workgroups for the parameters
};

// The wave's own LDS traffic in program order: the hardware keeps it, this keeps the compiler from moving it.
__device__ __forceinline__ void lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// log(1 + exp(v)) to relative precision on both sides: log1p(e) = 2 atanh(s), s = e / (2 + e) <= 1/3, and atanh(s) / s is a
// polynomial of degree 4 in s^2 (least squares over [0, 1/9]; off by 8e-9 of its value with these coefficients in f32).
// e = exp(-|v|).
__device__ __forceinline__ float softplus_f(float v, float e) {
    const float s = e * __builtin_amdgcn_rcpf(2.f + e), q = s * s;
    float p = 0.140873286f;
    p = p * q + 0.139807094f;
    p = p * q + 0.200124269f;
    p = p * q + 0.33333158f;
    p = p * q + 1.f;
    return fmaxf(v, 0.f) + 2.f * s * p;
}

// a log2 e.  -inf, a state that every token forgets, is the lowest number instead: tokens past a sequence's end have dt = 0 and
// leave it as it is
__device__ __forceinline__ float exponent_of(float a) {
    const float e = a * LOG2E;
    return e < -__FLT_MAX__ ? -__FLT_MAX__ : e;
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

// Each of four values summed over the 16 lanes of a row; lanes 4 k .. 4 k + 3 receive value sum16_of(k).  The first two steps
// halve the values as well as the lanes: a DPP add writes only the banks (groups of four lanes) of its mask, so two adds
// leave one value's sum in one half of the row and the other's in the other.  Eight adds in place of sixteen; the s_nops
// cover the two wait states between a VALU write and a DPP read of it.
__device__ __forceinline__ float sum16_four(float a, float b, float c, float d) {
    float p, q, s;
    asm("s_nop 1\n"
        "v_add_f32_dpp %0, %3, %3 row_ror:8 row_mask:0xf bank_mask:0x3\n"
        "v_add_f32_dpp %1, %5, %5 row_ror:8 row_mask:0xf bank_mask:0x3\n"
        "v_add_f32_dpp %0, %4, %4 row_ror:8 row_mask:0xf bank_mask:0xc\n"
        "v_add_f32_dpp %1, %6, %6 row_ror:8 row_mask:0xf bank_mask:0xc\n"
        "s_nop 0\n"
        "v_add_f32_dpp %2, %0, %0 row_half_mirror row_mask:0xf bank_mask:0x5\n"
        "v_add_f32_dpp %2, %1, %1 row_half_mirror row_mask:0xf bank_mask:0xa\n"
        "s_nop 1\n"
        "v_add_f32_dpp %2, %2, %2 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n"
        "s_nop 1\n"
        "v_add_f32_dpp %2, %2, %2 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
        : "=&v"(p), "=&v"(q), "=&v"(s) : "v"(a), "v"(b), "v"(c), "v"(d));
    return s;
}
__device__ __forceinline__ int sum16_of(int bank) { return (bank & 1) << 1 | bank >> 1; }
// A lane's NS values, one a state of its row, summed over the row's 16 lanes and put at s[4 rows x NS states]
template <int NS> __device__ __forceinline__ void put_sums(float* s, const float (&v)[NS], int r, int cl) {
    if constexpr (NS == 2) {
        const float a = sum16(v[0]), b = sum16(v[1]);
        s[r * 2 + (cl & 1)] = cl & 1 ? b : a;
    } else {
#pragma unroll
        for (int j = 0; j < NS; j += 4)
            s[r * NS + j + sum16_of(cl >> 2)] = sum16_four(v[j], v[j + 1], v[j + 2], v[j + 3]);
    }
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

// Where a wave is: its channels [c0, c0 + 16 CH) of group g up to the group's end (p0: the first one's place in a
// workspace), and its lane's places in both mappings.
template <typename T, int CH, int NS, int VE> struct Wave {
    static constexpr int WC = 16 * CH, NP = 4 * NS, NV = TT * WC / 64 / VE, SV = NS < 4 ? NS : 4;
    int lane, cl, r, g, c0, cend, p0;
    __device__ __forceinline__ Wave(const Args& A, int group, int first) {
        lane = threadIdx.x & 63;
        cl = lane & 15;
        r = lane >> 4;
        g = group;
        c0 = g * A.per + first;
        cend = (g + 1) * A.per;
        p0 = g * A.per_pad + first;
    }
    __device__ __forceinline__ int channel(int i) const { return c0 + cl * CH + i; }
    // staging: vector k of this lane is token trow(k) of the tile, channels c0 + tcol(k) ...
    __device__ __forceinline__ int trow(int k) const { return (k * 64 + lane) / (WC / VE); }
    __device__ __forceinline__ int tcol(int k) const { return (k * 64 + lane) % (WC / VE) * VE; }
    __device__ __forceinline__ int tat(int k) const { return trow(k) * WC + tcol(k); }
    __device__ __forceinline__ bool staged(int k, int v, int t0, int te) const {
        return t0 + trow(k) < te && c0 + tcol(k) + v < cend;
    }
    // A tile's base is uniform; 8 rows of any tensor span less than 2^31 bytes: the host sees to it.  there = false gives a
    // range of 0 bytes instead of a branch around the accesses: the hardware counts loads and stores in one order, and
    // behind a branch that may skip stores the compiler waits for them where it needs the loads before them (the forward of
    // 32 x 512 x 2048 keeping its states: 288 us with the branches, 238 without).
    __device__ __forceinline__ unsigned place(int k, int row, int t0, int te) const {
        return t0 + trow(k) < te && c0 + tcol(k) < cend ? (trow(k) * row + tcol(k)) * (unsigned)sizeof(T) : BUF_OUT;
    }
    __device__ __forceinline__ void fetch(const Rows& R, int b, int t0, int te, Raw<T, VE> (&v)[NV], bool there = true) const {
        const auto rs = buffer_of(static_cast<const T*>(R.p) + b * R.batch + t0 * R.row + c0, there ? BUF_BYTES : 0);
#pragma unroll
        for (int k = 0; k < NV; ++k) v[k] = buf_load<T, VE>(rs, place(k, (int)R.row, t0, te));
    }
    __device__ __forceinline__ void put(void* p, int b, int L, int D, int t0, int te, const Raw<T, VE> (&v)[NV]) const {
        const auto rs = buffer_of(static_cast<T*>(p) + ((long)b * L + t0) * D + c0, BUF_BYTES);
#pragma unroll
        for (int k = 0; k < NV; ++k) buf_store<T, VE>(rs, place(k, D, t0, te), v[k]);
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
                // (past the end not 0, whose product with an infinite dt is NaN: any finite dt gives a finite decay)
                a2[i][j] = channel(i) < cend && n < A.N ? exponent_of(A.a[(long)channel(i) * A.N + n]) : -1.2e-38f;
            }
    }
    // a state in its public layout [B][D][N].  (The lane is hidden from the compiler: these run once a sequence, and their
    // addresses and masks, known before the loop over tiles, would be kept in registers all through it.)
    __device__ __forceinline__ unsigned public_place(int l, int i, int j, int N) const {
        const int off = (l & 15) * CH + i, n = (l >> 4) * NS + j;
        return c0 + off < cend && n < N ? (unsigned)(off * N + n) * 4u : BUF_OUT;
    }
    __device__ __forceinline__ void load_public(const float* s, int b, int D, int N, float (&h)[CH][NS]) const {
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < NS; ++j) h[i][j] = 0.f;
        if (!s) return;
        int l = lane;
        asm volatile("" : "+v"(l));
        const auto rs = buffer_of(s + ((long)b * D + c0) * N, BUF_BYTES);
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < NS; ++j) h[i][j] = buf_load<float, 1>(rs, public_place(l, i, j, N)).get(0);
    }
    __device__ __forceinline__ void store_public(float* s, int b, int D, int N, const float (&h)[CH][NS]) const {
        int l = lane;
        asm volatile("" : "+v"(l));
        const auto rs = buffer_of(s + ((long)b * D + c0) * N, BUF_BYTES);
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                Raw<float, 1> f;
                f.set(0, h[i][j]);
                buf_store<float, 1>(rs, public_place(l, i, j, N), f);
            }
    }
    // ... and in a workspace: p = its first channel's place in it.  Channels past the end: 0, nothing
    __device__ __forceinline__ unsigned own_place(int i, int j) const {
        return channel(i) < cend ? (unsigned)((cl * CH + i) * NP + r * NS + j) * 4u : BUF_OUT;
    }
    __device__ __forceinline__ void load_own(const float* p, float (&h)[CH][NS]) const {
        const auto rs = buffer_of(p, BUF_BYTES);
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < NS; j += SV) {
                const Raw<float, SV> f = buf_load<float, SV>(rs, own_place(i, j));
#pragma unroll
                for (int q = 0; q < SV; ++q) h[i][j + q] = f.get(q);
            }
    }
    __device__ __forceinline__ void store_own(float* p, const float (&h)[CH][NS], bool there = true) const {
        const auto rs = buffer_of(p, there ? BUF_BYTES : 0);
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < NS; j += SV) {
                Raw<float, SV> f;
#pragma unroll
                for (int q = 0; q < SV; ++q) f.set(q, h[i][j + q]);
                buf_store<float, SV>(rs, own_place(i, j), f);
            }
    }
};

// b or c of a tile: element id = token * NP + state of [TT][NP], 0 past the tokens and the states.  The bits stay in a
// register each until they are used: two 16-bit values in an array would be packed into one register as soon as they are
// loaded, which waits for them where they were meant to be in flight.
template <typename T, int NP>
__device__ __forceinline__ unsigned fetch_shared(const Rows& R, int b, int t0, int te, int g, int N, int id) {
    const auto rs = buffer_of(static_cast<const T*>(R.p) + b * R.batch + t0 * R.row + (long)g * N, BUF_BYTES);
    const int t = id / NP, n = id % NP;
    const unsigned off = t0 + t < te && n < N ? (t * (int)R.row + n) * (unsigned)sizeof(T) : BUF_OUT;
    if constexpr (sizeof(T) == 4) return __builtin_amdgcn_raw_buffer_load_b32(rs, off, 0, 0);
    else return __builtin_amdgcn_raw_buffer_load_b16(rs, off, 0, 0);
}
template <typename T> __device__ __forceinline__ float shared_value(unsigned bits) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(bits);
    else return to_f32(__builtin_bit_cast(T, (unsigned short)bits));
}

// h is kept before every tile but the first (there it is the incoming state)
__host__ __device__ __forceinline__ int kept_tiles(int L) { return (L + TT - 1) / TT - 1; }
__device__ __forceinline__ int length_of(const Args& A, int b) {
    return A.lengths ? max(0, min(A.L, A.lengths[b])) : A.L;
}
// dt of staged raw values, 0 past the end (a token that moves no state); slope: its derivative, softplus' = sigmoid.  What
// a channel past the group's end has here is finite and meets only zeros.
template <bool SLOPE, typename W, typename R, int NV, int VE>
__device__ __forceinline__ void stage_steps(const W& w, const R (&d)[NV], const float* s_bias, int softplus, int t0, int te,
                                            float (&dt)[NV][VE], float (&slope)[NV][VE]) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int v = 0; v < VE; ++v) {
            dt[k][v] = d[k].get(v) + s_bias[w.tcol(k) + v];
            if (SLOPE) slope[k][v] = 1.f;
        }
    if (softplus) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int v = 0; v < VE; ++v) {
                const float u = dt[k][v], e = exp_f(-fabsf(u));
                dt[k][v] = softplus_f(u, e);
                if (SLOPE) slope[k][v] = (u < 0.f ? e : 1.f) * __builtin_amdgcn_rcpf(1.f + e);
            }
    }
    if (t0 + TT > te) {                                    // (the last tile of a sequence)
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int v = 0; v < VE; ++v)
                if (t0 + w.trow(k) >= te) dt[k][v] = 0.f;
    }
}

// The states past N, where N is not NP (PAD), have b = c = 0, and 0 times an infinite dt x or dcore would make NaN of a sum over
// states that is infinite.  In the forward a tile with such a value takes a second form of its loop, in which those states are
// kept at 0 (16383 tokens x 2048, N = 12, bf16: 147 us, 159 with a select or a mask per state in every tile, 145 without).  The
// backward has no registers for two forms and keeps their h and G at 0 by masks of bits (4 x 2048 x 2048, N = 12: 253 us; two
// forms 270, selects, whose conditions take scalar registers, 258, without 240).
struct Masked { static constexpr bool on = true; };
struct Plain { static constexpr bool on = false; };
__device__ __forceinline__ bool any_infinite(float largest) { return __any(largest == __builtin_inff()); }
template <bool PAD, int NS> struct Real {
    unsigned bits[NS];
    __device__ __forceinline__ Real(int r, int N) {
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            bits[j] = r * NS + j < N ? ~0u : 0u;
            if (PAD) asm volatile("" : "+v"(bits[j]));     // (a value, not a condition to the compiler)
        }
    }
    __device__ __forceinline__ float operator()(int j, float v) const {
        return PAD ? __uint_as_float(__float_as_uint(v) & bits[j]) : v;
    }
    // (what the first pass over a segment, which has no masks, left in their places of the workspace is not taken over)
    template <int CH> __device__ __forceinline__ void clear(float (&h)[CH][NS]) const {
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < NS; ++j) h[i][j] = (*this)(j, h[i][j]);
    }
};

// FULL: the forward.  Otherwise the first pass over a segment: its end state from 0, and sum dt.
template <typename T, int CH, int NS, int VE, bool FULL, bool PAD = false>
__global__ __launch_bounds__(64) void scan_fwd(Args A) {
    typedef Wave<T, CH, NS, VE> W;
    constexpr int NBC = TT * W::NP / 64;
    __shared__ __attribute__((aligned(16))) float s_dt[TT * W::WC], s_dtx[TT * W::WC], s_y[FULL ? TT * W::WC : 4],
        s_b[TT * W::NP], s_c[FULL ? TT * W::NP : 4], s_bias[W::WC], s_skip[FULL ? W::WC : 4];
    const int blks = A.fblk * A.G;
    const int blk = blockIdx.x % blks, seg = blockIdx.x / blks % A.segs, b = blockIdx.x / blks / A.segs;
    const W w(A, blk / A.fblk, blk % A.fblk * W::WC);
    const int len = length_of(A, b), ts = seg * A.seg_len, te = min(A.L, ts + A.seg_len), live = min(len, te);
    const long chans = (long)A.G * A.per_pad, at_seg = ((long)b * A.segs + seg) * chans + w.p0;
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
        if (A.segs > 1) {
            w.load_own(A.seg_h + at_seg * W::NP, h);
            Real<PAD, NS>(w.r, A.N).clear(h);
        } else w.load_public(A.state, b, A.D, A.N, h);
    }
    Raw<T, VE> x[W::NV], d[W::NV], z[W::NV], xn[W::NV], dn[W::NV];
    unsigned bn[NBC], cn[NBC];
    auto fetch = [&](int t0) {
        w.fetch(A.x, b, t0, live, xn);
        w.fetch(A.dt, b, t0, live, dn);
#pragma unroll
        for (int k = 0; k < NBC; ++k) {
            bn[k] = fetch_shared<T, W::NP>(A.b, b, t0, live, w.g, A.N, k * 64 + w.lane);
            if (FULL) cn[k] = fetch_shared<T, W::NP>(A.c, b, t0, live, w.g, A.N, k * 64 + w.lane);
        }
    };
    fetch(ts);
    for (int t0 = ts; t0 < live; t0 += TT) {
#pragma unroll
        for (int k = 0; k < W::NV; ++k) { x[k] = xn[k]; d[k] = dn[k]; }
        lds_order();                                       // (the last tile's reads are done)
        float step[W::NV][VE], largest = 0.f;
        stage_steps<false>(w, d, s_bias, A.flags & SOFTPLUS, t0, live, step, step);
#pragma unroll
        for (int k = 0; k < W::NV; ++k)
#pragma unroll
            for (int v = 0; v < VE; ++v) {
                const float dtx = step[k][v] * x[k].get(v);
                if (PAD) largest = fmaxf(largest, fabsf(dtx));
                s_dt[w.tat(k) + v] = step[k][v];
                s_dtx[w.tat(k) + v] = dtx;
            }
#pragma unroll
        for (int k = 0; k < NBC; ++k) {
            s_b[k * 64 + w.lane] = shared_value<T>(bn[k]);
            if (FULL) s_c[k * 64 + w.lane] = shared_value<T>(cn[k]);
        }
        lds_order();
        if (FULL) w.fetch(A.gate, b, t0, live, z, A.gate.p != nullptr);
        fetch(t0 + TT);                                    // (past the end: zeros)
        if (FULL) w.store_own(A.keep + (((long)b * kept_tiles(A.L) + t0 / TT - 1) * chans + w.p0) * W::NP, h, A.keep && t0 > 0);
        auto tokens = [&](auto form) {
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
                        // (which product is rounded before the sum is not left to the compiler: its choice differed between forms)
                        h[i][j] = __builtin_fmaf(dtx[i], bv[j], __builtin_amdgcn_exp2f(dt[i] * a2[i][j]) * h[i][j]);
                        if (decltype(form)::on && w.r * NS + j >= A.N) h[i][j] = 0.f;
                        if (FULL) y[i] += h[i][j] * cv[j];
                    }
                }
                if (FULL) s_y[t * W::WC + w.cl * CH + own_channel<CH>(w.r)] = sum_states<CH>(y);
            }
        };
        if (PAD && any_infinite(largest)) tokens(Masked()); else tokens(Plain());
        if (FULL) {
            lds_order();
#pragma unroll
            for (int k = 0; k < W::NV; ++k)
#pragma unroll
                for (int v = 0; v < VE; ++v) step[k][v] = s_y[w.tat(k) + v];
            if (A.flags & SKIP) {                          // (not 0 times an x that may be infinite)
#pragma unroll
                for (int k = 0; k < W::NV; ++k)
#pragma unroll
                    for (int v = 0; v < VE; ++v) step[k][v] += s_skip[w.tcol(k) + v] * x[k].get(v);
            }
            if (A.gate.p) {
#pragma unroll
                for (int k = 0; k < W::NV; ++k)
#pragma unroll
                    for (int v = 0; v < VE; ++v) step[k][v] *= silu_f(z[k].get(v));
            }
#pragma unroll
            for (int k = 0; k < W::NV; ++k) {
#pragma unroll
                for (int v = 0; v < VE; ++v) d[k].set(v, step[k][v]);
                if (t0 + TT > len && t0 + w.trow(k) >= len) d[k].zero();
            }
            w.put(A.y, b, A.L, A.D, t0, te, d);
        }
    }
    if (FULL) {
        for (int t0 = live > ts ? ts + (live - ts + TT - 1) / TT * TT : ts; t0 < te; t0 += TT) {     // past the end: zero rows
#pragma unroll
            for (int k = 0; k < W::NV; ++k) x[k].zero();
            w.put(A.y, b, A.L, A.D, t0, te, x);
        }
        if (A.last && seg == A.segs - 1) w.store_public(A.last, b, A.D, A.N, h);
    } else {
        w.store_own(A.seg_h + at_seg * W::NP, h);
        if (w.r == 0) {
#pragma unroll
            for (int i = 0; i < CH; ++i)
                if (w.channel(i) < w.cend) A.seg_dt[at_seg + w.cl * CH + i] = sum_dt[i];
        }
    }
}

// Chains the segments: seg_h[s] becomes the state (REV: the adjoint) that comes into segment s.  One thread a state, and it
// is bound by the latency of its loads (a few segments' states of 2048 x 16 are a few hundred KB): CHAIN of them in flight.
constexpr int CHAIN = 32;
template <int NP, bool REV> __global__ __launch_bounds__(256) void scan_chain(Args A) {
    const long chans = (long)A.G * A.per_pad, id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= A.B * chans * NP) return;
    const int n = (int)(id % NP), p = (int)(id / NP % chans), b = (int)(id / NP / chans);
    const int g = p / A.per_pad, off = p % A.per_pad, c = g * A.per + off;
    if (off >= A.per || n >= A.N) return;
    const float* start = REV ? A.dlast : A.state;
    const float a = exponent_of(A.a[(long)c * A.N + n]);
    float h = start ? start[((long)b * A.D + c) * A.N + n] : 0.f;
    const long first = (long)b * A.segs * chans + p;
    float* q = A.seg_h + first * NP + n;
    const float* dt = A.seg_dt + first;
    for (int s0 = 0; s0 < A.segs; s0 += CHAIN) {
        float e[CHAIN], d[CHAIN];
#pragma unroll
        for (int u = 0; u < CHAIN; ++u) {
            const int s = REV ? max(A.segs - 1 - s0 - u, 0) : min(s0 + u, A.segs - 1);
            e[u] = q[s * chans * NP];
            d[u] = dt[s * chans];
        }
#pragma unroll
        for (int u = 0; u < CHAIN; ++u) {
            const int s = REV ? A.segs - 1 - s0 - u : s0 + u;
            if (s >= 0 && s < A.segs) {
                q[s * chans * NP] = h;
                // (a segment's whole decay may underflow where no token's does, and an infinite state stays infinite)
                const float decay = __builtin_amdgcn_exp2f(d[u] * a);
                h = __builtin_fmaf(decay < 0x1p-149f ? 0x1p-149f : decay, h, e[u]);
            }
        }
    }
}

// The backward's first pass over a segment: the adjoint that leaves it at its front when 0 comes in at its end.
template <typename T, int CH, int NS, int VE>
__global__ __launch_bounds__(64) void scan_bwd_ends(Args A) {
    typedef Wave<T, CH, NS, VE> W;
    constexpr int NBC = TT * W::NP / 64;
    __shared__ __attribute__((aligned(16))) float s_dt[TT * W::WC], s_g[TT * W::WC], s_c[TT * W::NP], s_bias[W::WC];
    const int blks = A.fblk * A.G;
    const int blk = blockIdx.x % blks, seg = blockIdx.x / blks % A.segs, b = blockIdx.x / blks / A.segs;
    const W w(A, blk / A.fblk, blk % A.fblk * W::WC);
    const int ts = seg * A.seg_len, te = min(length_of(A, b), min(A.L, ts + A.seg_len));
    const long chans = (long)A.G * A.per_pad, at_seg = ((long)b * A.segs + seg) * chans + w.p0;
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
    unsigned cn[NBC];
    auto fetch = [&](int t0) {
        w.fetch(A.dt, b, t0, te, dn);
        if (A.gate.p) w.fetch(A.gate, b, t0, te, zn);
        w.fetch(A.dy, b, t0, te, gn);
#pragma unroll
        for (int k = 0; k < NBC; ++k) cn[k] = fetch_shared<T, W::NP>(A.c, b, t0, te, w.g, A.N, k * 64 + w.lane);
    };
    int t0 = ts + (te - ts - 1) / TT * TT;
    if (te > ts) fetch(t0);
    for (; te > ts && t0 >= ts; t0 -= TT) {
        lds_order();
        float step[W::NV][VE], dcore[W::NV][VE];
        stage_steps<false>(w, dn, s_bias, A.flags & SOFTPLUS, t0, te, step, step);
#pragma unroll
        for (int k = 0; k < W::NV; ++k)
#pragma unroll
            for (int v = 0; v < VE; ++v) dcore[k][v] = gn[k].get(v);
        if (A.gate.p) {
#pragma unroll
            for (int k = 0; k < W::NV; ++k)
#pragma unroll
                for (int v = 0; v < VE; ++v) dcore[k][v] *= silu_f(zn[k].get(v));
        }
#pragma unroll
        for (int k = 0; k < W::NV; ++k)
#pragma unroll
            for (int v = 0; v < VE; ++v) {
                s_dt[w.tat(k) + v] = step[k][v];
                s_g[w.tat(k) + v] = dcore[k][v];
            }
#pragma unroll
        for (int k = 0; k < NBC; ++k) s_c[k * 64 + w.lane] = shared_value<T>(cn[k]);
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
    w.store_own(A.seg_h + at_seg * W::NP, g);
    if (w.r == 0) {
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (w.channel(i) < w.cend) A.seg_dt[at_seg + w.cl * CH + i] = sum_dt[i];
    }
}

// The backward.  Tiles from the last to the first; inside a tile the states are computed again from the kept one, forwards,
// staying in registers (h before each of the TT tokens), then the adjoint runs backwards over them.  Those TT CH NS
// registers are why a lane has half the forward's channels: at 16 states a lane they do not fit, and the spills cost more
// than all the rest (566 us against 88 of the forward at 4 x 2048 tokens x 2048 channels, N = 16, bf16; this form: 231).  What
// two waves a SIMD leave of 256 registers keeps the decays of a tile's last KD tokens for the way back (five: 251 -> 231 us;
// with a sixth one wave fits, 308 us); the other tokens' are formed again.  The scalar registers do not suffice: about 100 of
// them lie in lanes of vector registers, and every tile reads them back on the vector ALU, which is busy 3/4 of the time.
// The BW waves of a workgroup take neighbouring channels, share b and c in LDS and join their sums db, dc over channels
// there: part_bc[workgroup of the group][B][L][G][2][N].  A workgroup takes the sequences of its batch group one after the
// other, so that its sums over tokens leave once: part_p[(batch group, segment)]{da [channel][NP], dskip, ddt_bias}.
template <typename T, int CH, int NS, int VE, bool PAD>
__global__ __launch_bounds__(64 * BW, CH * NS > 8 ? 1 : 2) void scan_bwd(Args A) {
    typedef Wave<T, CH, NS, VE> W;
    constexpr int TILE = TT * W::WC, SH = TT * W::NP, NBC = (2 * SH + 64 * BW - 1) / (64 * BW), 
                  KD = CH * NS > 8 ? 0 : CH * NS < 8 || CH == 1 || (VE > 1 && sizeof(T) == 2) ? 5 : VE > 1 ? 2 : 0;
    __shared__ __attribute__((aligned(16))) float lds[BW][6 * TILE + 2 * W::WC], s_bc[2 * SH], s_part[BW][2 * SH];
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int blks = A.bblk * A.G;
    const int blk = blockIdx.x % blks, seg = blockIdx.x / blks % A.segs, group = blockIdx.x / blks / A.segs;
    const W w(A, blk / A.bblk, (blk % A.bblk * BW + wv) * W::WC);
    const bool live = w.c0 < w.cend;                       // (a wave past the group's end only keeps step)
    float *s_dt = lds[wv], *s_dtx = s_dt + TILE, *s_g = s_dtx + TILE, *s_y = s_g + TILE, *s_gt = s_y + TILE,
          *s_bias = s_gt + 2 * TILE, *s_skip = s_bias + W::WC, *s_db = s_part[wv], *s_dc = s_db + SH;
    const float *s_b = s_bc, *s_c = s_bc + SH;
    const long chans = (long)A.G * A.per_pad;
    const int ts = seg * A.seg_len, tend = min(A.L, ts + A.seg_len);
    const Real<PAD, NS> real(w.r, A.N);
    // (without a skip its 0 meets no infinity.  A mask in a vector register: a branch here costs 3 % of the kernel)
    unsigned skip_bits = A.flags & SKIP ? ~0u : 0u;
    asm volatile("" : "+v"(skip_bits));
    auto if_skip = [&](float v) { return __uint_as_float(__float_as_uint(v) & skip_bits); };
    float a2[CH][NS], g[CH][NS], da[CH][NS], sum_skip[W::NV][VE], sum_bias[W::NV][VE];
    w.lane_a(A, a2);
    w.stage_param(A.dt_bias, s_bias);
    w.stage_param(A.skip, s_skip);
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int j = 0; j < NS; ++j) da[i][j] = 0.f;
#pragma unroll
    for (int k = 0; k < W::NV; ++k)
#pragma unroll
        for (int v = 0; v < VE; ++v) sum_skip[k][v] = sum_bias[k][v] = 0.f;
    if (!live)
        for (int k = w.lane; k < 2 * SH; k += 64) s_db[k] = 0.f;
    // what the next tile needs, in flight while this one is worked on: of this sequence, or of the batch group's next one
    // that has tokens in this segment
    Raw<T, VE> xn[W::NV], dn[W::NV], zn[W::NV], gn[W::NV];
    unsigned sn[NBC];
    float hn[CH][NS];
    auto last_tile = [&](int b) {
        const int n = min(length_of(A, b), tend) - ts;
        return n > 0 ? ts + (n - 1) / TT * TT : -1;
    };
    auto fetch = [&](int b, int t0) {
        const int te = min(length_of(A, b), tend);
        w.fetch(A.x, b, t0, te, xn);
        w.fetch(A.dt, b, t0, te, dn);
        if (A.gate.p) w.fetch(A.gate, b, t0, te, zn);
        w.fetch(A.dy, b, t0, te, gn);
#pragma unroll
        for (int k = 0; k < NBC; ++k) {
            const int id = k * 64 * BW + threadIdx.x;
            sn[k] = fetch_shared<T, W::NP>(id < SH ? A.b : A.c, b, t0, id < 2 * SH ? te : t0, w.g, A.N, id % SH);
        }
        if (t0 > 0) w.load_own(A.keep + (((long)b * kept_tiles(A.L) + t0 / TT - 1) * chans + w.p0) * W::NP, hn);
        else w.load_public(A.state, b, A.D, A.N, hn);
    };
    auto fetch_next = [&](int b) {                         // the first tile to come of sequence b or a later one
        for (; b < A.B; b += A.bgroups)
            if (last_tile(b) >= 0) { fetch(b, last_tile(b)); return; }
    };
    fetch_next(group);
    for (int b = group; b < A.B; b += A.bgroups) {
        const int te = min(length_of(A, b), tend), t_last = last_tile(b);
        for (int t0 = t_last < 0 ? ts : t_last + TT; t0 < tend; t0 += TT) {      // past the end of this sequence: zero rows
            Raw<T, VE> x[W::NV];
#pragma unroll
            for (int k = 0; k < W::NV; ++k) x[k].zero();
            w.put(A.dx, b, A.L, A.D, t0, tend, x);
            w.put(A.ddt, b, A.L, A.D, t0, tend, x);
            if (A.gate.p) w.put(A.dgate, b, A.L, A.D, t0, tend, x);
        }
        if (A.segs > 1) {
            w.load_own(A.seg_h + (((long)b * A.segs + seg) * chans + w.p0) * W::NP, g);
            real.clear(g);
        } else w.load_public(A.dlast, b, A.D, A.N, g);
        for (int t0 = t_last; t0 >= ts; t0 -= TT) {
            Raw<T, VE> x[W::NV], d[W::NV], z[W::NV], gy[W::NV];
            float hist[TT][CH][NS], h[CH][NS], kd[KD > 0 ? KD : 1][CH][NS];
#pragma unroll
            for (int k = 0; k < W::NV; ++k) { x[k] = xn[k]; d[k] = dn[k]; z[k] = zn[k]; gy[k] = gn[k]; }
#pragma unroll
            for (int i = 0; i < CH; ++i)
#pragma unroll
                for (int j = 0; j < NS; ++j) h[i][j] = hn[i][j];
#pragma unroll
            for (int k = 0; k < NBC; ++k)
                if (k * 64 * BW + (int)threadIdx.x < 2 * SH) s_bc[k * 64 * BW + threadIdx.x] = shared_value<T>(sn[k]);
            float step[W::NV][VE], slope[W::NV][VE], sig[W::NV][VE], dcore[W::NV][VE];
            if (live) {
                stage_steps<true>(w, d, s_bias, A.flags & SOFTPLUS, t0, te, step, slope);
#pragma unroll
                for (int k = 0; k < W::NV; ++k)
#pragma unroll
                    for (int v = 0; v < VE; ++v) dcore[k][v] = gy[k].get(v);
                if (A.gate.p) {
#pragma unroll
                    for (int k = 0; k < W::NV; ++k)
#pragma unroll
                        for (int v = 0; v < VE; ++v) {
                            sig[k][v] = sigmoid_f(z[k].get(v));
                            dcore[k][v] *= z[k].get(v) * sig[k][v];
                        }
                }
#pragma unroll
                for (int k = 0; k < W::NV; ++k)
#pragma unroll
                    for (int v = 0; v < VE; ++v) {
                        s_dt[w.tat(k) + v] = step[k][v];
                        s_dtx[w.tat(k) + v] = step[k][v] * x[k].get(v);
                        s_g[w.tat(k) + v] = dcore[k][v];
                    }
            }
            __syncthreads();                               // b, c are there; the last tile's s_part has been read
            if (t0 > ts) fetch(b, t0 - TT); else fetch_next(b + A.bgroups);
            if (live) {
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
                            const float decay = __builtin_amdgcn_exp2f(dt[i] * a2[i][j]);
                            if (t >= TT - KD) kd[t >= TT - KD ? t - (TT - KD) : 0][i][j] = decay;
                            h[i][j] = real(j, __builtin_fmaf(decay, h[i][j], dtx[i] * bv[j]));
                            y[i] += h[i][j] * cv[j];
                            sc[j] += h[i][j] * dc[i];
                        }
                    }
                    s_y[t * W::WC + w.cl * CH + own_channel<CH>(w.r)] = sum_states<CH>(y);
                    put_sums<NS>(s_dc + t * W::NP, sc, w.r, w.cl);
                }
                // a token past the end takes no part in da: its dt of 0 times an infinite state would be NaN.  (The empty asm
                // keeps this a branch over the tokens that are there, not a select for each of their states.)
#pragma unroll
                for (int t = 1; t < TT; ++t)
                    if (t0 + t >= te) {
                        asm volatile("");
#pragma unroll
                        for (int i = 0; i < CH; ++i)
#pragma unroll
                            for (int j = 0; j < NS; ++j) hist[t][i][j] = 0.f;
                    }
                lds_order();                           // (and the decays are formed again, not held in registers)
#pragma unroll
                for (int t = TT - 1; t >= 0; --t) {
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
                            const float G = real(j, g[i][j] + dc[i] * cv[j]);
                            gb[i] += G * bv[j];
                            sb[j] += G * dtx[i];
                            g[i][j] = G * (t >= TT - KD ? kd[t >= TT - KD ? t - (TT - KD) : 0][i][j]
                                                        : __builtin_amdgcn_exp2f(dt[i] * a2[i][j]));
                            const float th = g[i][j] * hist[t][i][j];
                            ta[i] += th * a2[i][j];
                            da[i][j] += th * dt[i];
                        }
                    }
                    // both sums over states at once: even rows receive gb's, odd rows ta's
                    float both;
                    if constexpr (CH == 2) both = swap_add16(swap_add32(gb[0], gb[1]), swap_add32(ta[0], ta[1]));
                    else both = swap_add16(swap_add32(gb[0], gb[0]), swap_add32(ta[0], ta[0]));
                    s_gt[(w.r & 1) * TILE + t * W::WC + w.cl * CH + (CH == 2 ? w.r >> 1 : 0)] = both;
                    put_sums<NS>(s_db + t * W::NP, sb, w.r, w.cl);
                }
                lds_order();
                if (A.gate.p) {
#pragma unroll
                    for (int k = 0; k < W::NV; ++k) {
#pragma unroll
                        for (int v = 0; v < VE; ++v) {
                            const float core = s_y[w.tat(k) + v] + s_skip[w.tcol(k) + v] * if_skip(x[k].get(v));
                            z[k].set(v, gy[k].get(v) * core * sig[k][v] * (1.f + z[k].get(v) * (1.f - sig[k][v])));
                        }
                        if (t0 + TT > te && t0 + w.trow(k) >= te) z[k].zero();
                    }
                    w.put(A.dgate, b, A.L, A.D, t0, tend, z);
                }
#pragma unroll
                for (int k = 0; k < W::NV; ++k) {
                    const bool past = t0 + TT > te && t0 + w.trow(k) >= te;
#pragma unroll
                    for (int v = 0; v < VE; ++v) {
                        const float gb = s_gt[w.tat(k) + v], xv = x[k].get(v);
                        float dr = (s_gt[TILE + w.tat(k) + v] * LN2 + xv * gb) * slope[k][v];
                        if (past) dr = 0.f;
                        sum_bias[k][v] += dr;
                        sum_skip[k][v] += past ? 0.f : dcore[k][v] * xv;
                        d[k].set(v, dr);
                        x[k].set(v, __builtin_fmaf(step[k][v], gb, s_skip[w.tcol(k) + v] * if_skip(dcore[k][v])));
                    }
                    if (past) x[k].zero();
                }
                w.put(A.dx, b, A.L, A.D, t0, tend, x);
                w.put(A.ddt, b, A.L, A.D, t0, tend, d);
            }
            __syncthreads();                               // every wave's s_db, s_dc are there; b and c have been read
            const auto rs = buffer_of(
                A.part_bc + ((((long)(blk % A.bblk) * A.B + b) * A.L + t0) * A.G + w.g) * 2 * A.N, BUF_BYTES);
#pragma unroll
            for (int k = 0; k < NBC; ++k) {
                const int id = k * 64 * BW + threadIdx.x, t = id % SH / W::NP, n = id % W::NP;
                if (id >= 2 * SH) break;
                float s = 0.f;
#pragma unroll
                for (int u = 0; u < BW; ++u) s += s_part[u][id];
                __builtin_amdgcn_raw_buffer_store_b32(
                    __float_as_uint(s), rs,
                    t0 + t < te && n < A.N ? ((t * A.G * 2 + (id < SH ? 0 : 1)) * A.N + n) * 4u : BUF_OUT, 0, 0);
            }
        }
        if (A.dstate && seg == 0) w.store_public(A.dstate, b, A.D, A.N, g);
    }
    if (!live) return;                                     // (no barrier follows)
    float* out = A.part_p + ((long)group * A.segs + seg) * chans * (W::NP + 2);
    w.store_own(out + (long)w.p0 * W::NP, da);
    // sums over the tokens of a tile: lanes that staged the same channels meet in LDS
    for (int half = 0; half < 2; ++half) {
        lds_order();
#pragma unroll
        for (int k = 0; k < W::NV; ++k)
#pragma unroll
            for (int v = 0; v < VE; ++v) s_dt[w.tat(k) + v] = half ? sum_bias[k][v] : sum_skip[k][v];
        lds_order();
        if (w.lane < W::WC && w.c0 + w.lane < w.cend) {
            float s = 0.f;
#pragma unroll
            for (int t = 0; t < TT; ++t) s += s_dt[t * W::WC + w.lane];
            out[chans * (W::NP + half) + w.p0 + w.lane] = s;
        }
    }
}

// part_p's rows summed in a fixed order (16 row lanes x 64 columns) and put in their public places.
template <int NP>
__device__ __forceinline__ void sum_params(const float* __restrict__ part, int rows, int per, int per_pad, int N, int G,
                                           float* __restrict__ da, float* __restrict__ dskip, float* __restrict__ dbias) {
    const long chans = (long)G * per_pad, cols = chans * (NP + 2), col = (long)blockIdx.x * 64 + (threadIdx.x & 63);
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
    const bool is_a = col < chans * NP;
    const long p = is_a ? col / NP : (col - chans * NP) % chans;
    if (p % per_pad >= per) return;                        // (a place between two groups)
    const long c = p / per_pad * per + p % per_pad;
    if (is_a) {
        if (col % NP < N) da[c * N + col % NP] = t;
    } else if (col < chans * (NP + 1)) {
        if (dskip) dskip[c] = t;
    } else if (dbias) dbias[c] = t;
}

// db and dc: the channel blocks' shares in a fixed order; rows past a sequence's length are 0.  Each share is read once, eight
// in flight a thread.  Workgroup `block` of `blocks`.
template <typename T>
__device__ __forceinline__ void sum_shared(const float* __restrict__ part, const int* __restrict__ lengths, int B, int L, int G,
                                           int N, int nblk, T* __restrict__ db, T* __restrict__ dc, int block, int blocks) {
    const long n = (long)B * L * G * 2 * N;
    const int w = G * 2 * N;                               // values a token
    for (long id0 = (long)block * 1024; id0 < n; id0 += (long)blocks * 1024) {
        const long id = id0 + threadIdx.x;
        if (id >= n) return;
        // (the divisions of 64 bits are the workgroup's, a thread's are of 32)
        const long tok0 = id0 / w, seq0 = tok0 / L;
        const unsigned r = (unsigned)(id0 - tok0 * w) + threadIdx.x, t = (unsigned)(tok0 - seq0 * L) + r / w;
        float s = 0.f;
        if (!lengths || (int)(t % (unsigned)L) < lengths[seq0 + t / (unsigned)L]) {
#pragma unroll 8
            for (int k = 0; k < nblk; ++k) s += part[k * n + id];
        }
        const unsigned v = r % w, g = v / (2u * N), e = v % (2u * N);
        const long row = (tok0 + r / w) * G + g;
        (e < (unsigned)N ? db[row * N + e] : dc[row * N + e - N]) = from_f32<T>(s);
    }
}

// Both in one launch, the first A.params workgroups for the parameters: each is a few microseconds of waiting for its loads
// (4 x 2048 x 2048 9.9 us, 5.8 + 5.7 in two launches; 256 x 14 x 2048 7.3, 4.2 + 5.4).
template <typename T, int NP> __global__ __launch_bounds__(1024) void scan_join(Args A) {
    const int block = blockIdx.x;
    if (block < A.params)
        sum_params<NP>(A.part_p, A.bgroups * A.segs, A.per, A.per_pad, A.N, A.G, A.da, A.dskip, A.dbias);
    else
        sum_shared<T>(A.part_bc, A.lengths, A.B, A.L, A.G, A.N, A.bblk, static_cast<T*>(A.db), static_cast<T*>(A.dc),
                      block - A.params, (int)gridDim.x - A.params);
}

// One token: a lane takes four states of a channel, LN lanes a channel, 256 / LN channels of one sequence a workgroup.  Bound
// by the state's bytes, read and written once.
template <typename T, int LN, bool VEC>
__global__ __launch_bounds__(256) void scan_token(Rows x, float* __restrict__ state, long state_batch, Rows dt, Rows gate,
                                                  Rows b, Rows c, const float* __restrict__ a,
                                                  const float* __restrict__ skip, const float* __restrict__ dt_bias,
                                                  int softplus, int D, int N, int per, int blocks, T* __restrict__ y) {
    const int bi = blockIdx.x / blocks, d = (blockIdx.x - bi * blocks) * (256 / LN) + threadIdx.x / LN;
    const int part = threadIdx.x % LN, n0 = part * 4;
    if (d >= D) return;                                    // (whole channels: the LN lanes stay together)
    const long shared = per == D ? 0 : (long)(d / per) * N;
    const T* bp = static_cast<const T*>(b.p) + bi * b.batch + shared;
    const T* cp = static_cast<const T*>(c.p) + bi * c.batch + shared;
    float* hp = state + bi * state_batch + (long)d * N;
    Raw<float, 4> h, av;
    Raw<T, 4> bv, cv;
    h.zero();
    av.zero();
    bv.zero();
    cv.zero();
    if constexpr (VEC) {
        if (n0 < N) {
            h.load(hp + n0);
            av.load(a + (long)d * N + n0);
            bv.load(bp + n0);
            cv.load(cp + n0);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (n0 + k < N) {
                h.v[k] = hp[n0 + k];
                av.v[k] = a[(long)d * N + n0 + k];
                bv.v[k] = bp[n0 + k];
                cv.v[k] = cp[n0 + k];
            }
    }
    const float xv = to_f32(static_cast<const T*>(x.p)[bi * x.batch + d]);
    const float zv = gate.p ? to_f32(static_cast<const T*>(gate.p)[bi * gate.batch + d]) : 0.f;
    const float sk = skip ? skip[d] : 0.f;
    float step = to_f32(static_cast<const T*>(dt.p)[bi * dt.batch + d]) + (dt_bias ? dt_bias[d] : 0.f);
    if (softplus) step = softplus_f(step, exp_f(-fabsf(step)));
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        // (a state past N stays 0 whatever dt and x are)
        h.v[k] = n0 + k < N ? exp_f(step * av.v[k]) * h.v[k] + step * xv * bv.get(k) : 0.f;
        s += h.v[k] * cv.get(k);
    }
    if constexpr (VEC) {
        if (n0 < N) h.store(hp + n0);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (n0 + k < N) hp[n0 + k] = h.v[k];
    }
#pragma unroll
    for (int o = 1; o < LN; o <<= 1) s += __shfl_xor(s, o);
    if (part == 0) {
        if (skip) s += sk * xv;
        if (gate.p) s *= silu_f(zv);
        y[(long)bi * D + d] = from_f32<T>(s);
    }
}

// Padded states, and channels of a forward wave and of a backward workgroup.
int np_of(int N) { return N <= 8 ? 8 : N <= 16 ? 16 : N <= 32 ? 32 : 64; }
int fwd_channels(int N) { return N <= 16 ? 64 : N <= 32 ? 32 : 16; }
int bwd_channels(int N) { return N <= 16 ? 32 * BW : 16 * BW; }

// Segments cost a second pass over the tokens, so there are none while whole sequences make enough waves (counted as the
// forward's: of 64 channels up to 16 states, 32 up to 32, 16 above; the figures are of 16 states): 400 in the forward
// (B x 512 x 2048: 512 waves 122 us and 162 in segments, 384 118 and 124, 256 115 and 90), 640 in the backward (768 waves 446
// us and 472, 512 335 and 316).  Below that, enough for 4096 waves with eight tiles
// each at least (2048 to 8192 waves are the same within 3 %), or for 1024 waves with two tiles each, whichever is more
// (3 x 577 x 600, 30 waves whole, training: 145 us with eight tiles each, 101 with four, 82 with two).
void plan(Args& A, bool bwd) {
    A.per = A.D / A.G;
    A.fblk = (A.per + fwd_channels(A.N) - 1) / fwd_channels(A.N);
    A.bblk = (A.per + bwd_channels(A.N) - 1) / bwd_channels(A.N);
    // Workspaces hold a group's channels as whole backward workgroups take them, which costs little with one group.  Narrow
    // groups, of which there may be many, are held as they are (64 x 4096 tokens, 64 channels in 4 groups: the kept states
    // would take 1.07 GB in place of 134 MB).
    A.per_pad = A.bblk * bwd_channels(A.N);
    if (A.G > 1 && 4 * A.per < A.per_pad) A.per_pad = A.per;
    const long waves = (long)A.B * A.G * A.fblk;
    long s = 1;
    if (waves < (bwd ? 640 : 400)) {
        s = std::min(4096 / waves, (long)A.L / (8 * TT));
        s = std::max(s, std::min(1024 / waves, (long)A.L / (2 * TT)));
        s = std::max(s, 1L);
    }
    long len = (A.L + s - 1) / s;
    len = (len + TT - 1) / TT * TT;
    A.seg_len = (int)len;
    A.segs = (int)((A.L + len - 1) / len);
    // whole sequences in few waves: half the channels a wave, twice the waves (32 x 512 x 2048: 168 us, 190 without; at 4096
    // waves no difference)
    A.narrow = A.segs == 1 && waves < 4096 && A.N <= 32;
    if (A.narrow) A.fblk = (A.per + fwd_channels(A.N) / 2 - 1) / (fwd_channels(A.N) / 2);
    // the backward's sums over tokens leave a workgroup once: as few workgroups as still fill the chip
    const long g = 1024 / ((long)A.G * A.bblk * A.segs);
    A.bgroups = (int)(g < 1 ? 1 : g > A.B ? A.B : g);
}

bool bad_shape(int dtype, int B, int L, int D, int N, int G) {
    return !vqa_dtype_ok(dtype) || B < 1 || L < 1 || L > 0x3fffffff || D < 1 || N < 1 || N > 64 || G < 1 || D % G != 0 ||
           (double)B * L > 1e9 || (double)B * L * D > 4e11 || (double)B * D > 1e9 || (double)B * L * G * N > 1e11 ||
           (double)G * (D / G + 128) * B > 2e9 || (double)G * (D / G + 128) * (np_of(N) + 2) > 2.4e8 ||
           // (a grid has fewer than 2^32 threads: the forward's waves.  Segments and half waves are for few of them.)
           (double)B * G * ((D / G + fwd_channels(N) - 1) / fwd_channels(N)) * 64 > 4.29e9;
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

// Workspaces, in floats: the segments' states and sums of dt (none without segments), the backward's partial sums
// (each a multiple of 16 bytes)
long whole(long floats) { return (floats + 3) / 4 * 4; }
long seg_floats(const Args& A) {
    return A.segs > 1 ? whole((long)A.B * A.segs * A.G * A.per_pad * (np_of(A.N) + 1)) : 0;
}
float* seg_dt_of(const Args& A, float* ws) { return ws + (long)A.B * A.segs * A.G * A.per_pad * np_of(A.N); }
long part_p_floats(const Args& A) { return whole((long)A.bgroups * A.segs * A.G * A.per_pad * (np_of(A.N) + 2)); }
long part_bc_floats(const Args& A) { return (long)A.bblk * A.B * A.L * A.G * 2 * A.N; }

template <int NP, bool REV> int chain(const Args& A, hipStream_t st) {
    const long n = (long)A.B * A.G * A.per_pad * NP;
    scan_chain<NP, REV><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(A);
    CHECK_LAUNCH();
    return VQA_OK;
}

// CH, VE: the forward's channels a lane and elements a load; BCH, BVE: the backward's
template <typename T, int NS, int CH, int VE, int BCH, int BVE, bool PAD> int launch(bool bwd, const Args& A, hipStream_t st) {
    const unsigned waves = (unsigned)((long)A.fblk * A.G * A.segs * A.B);
    int rc = VQA_OK;
    if (A.segs > 1) {
        if (bwd) scan_bwd_ends<T, CH, NS, VE><<<waves, 64, 0, st>>>(A);
        else scan_fwd<T, CH, NS, VE, false><<<waves, 64, 0, st>>>(A);
        CHECK_LAUNCH();
        rc = bwd ? chain<4 * NS, true>(A, st) : chain<4 * NS, false>(A, st);
        if (rc != VQA_OK) return rc;
    }
    if constexpr (CH > 1)
        if (!bwd && A.narrow) {
            scan_fwd<T, CH / 2, NS, (VE < CH ? VE : CH), true, PAD><<<waves, 64, 0, st>>>(A);
            CHECK_LAUNCH();
            return VQA_OK;
        }
    if (!bwd) {
        scan_fwd<T, CH, NS, VE, true, PAD><<<waves, 64, 0, st>>>(A);
        CHECK_LAUNCH();
        return VQA_OK;
    }
    scan_bwd<T, BCH, NS, BVE, PAD><<<(unsigned)((long)A.bblk * A.G * A.segs * A.bgroups), 64 * BW, 0, st>>>(A);
    CHECK_LAUNCH();
    const long shared = std::min(((long)A.B * A.L * A.G * 2 * A.N + 1023) / 1024, 16384L);
    scan_join<T, 4 * NS><<<(unsigned)(A.params + shared), 1024, 0, st>>>(A);
    CHECK_LAUNCH();
    return VQA_OK;
}
template <typename T, bool PAD> int by_states(bool bwd, bool vec, const Args& A, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    if (A.N <= 8) return vec ? launch<T, 2, 4, V, 2, 4, PAD>(bwd, A, st) : launch<T, 2, 4, 1, 2, 1, PAD>(bwd, A, st);
    if (A.N <= 16) return vec ? launch<T, 4, 4, V, 2, 4, PAD>(bwd, A, st) : launch<T, 4, 4, 1, 2, 1, PAD>(bwd, A, st);
    if (A.N <= 32) return vec ? launch<T, 8, 2, 4, 1, 2, PAD>(bwd, A, st) : launch<T, 8, 2, 1, 1, 1, PAD>(bwd, A, st);
    return vec ? launch<T, 16, 1, 2, 1, 2, PAD>(bwd, A, st) : launch<T, 16, 1, 1, 1, 1, PAD>(bwd, A, st);
}
template <typename T> int by_states(bool bwd, bool vec, const Args& A, hipStream_t st) {
    return A.N == np_of(A.N) ? by_states<T, false>(bwd, vec, A, st) : by_states<T, true>(bwd, vec, A, st);
}
int by_type(bool bwd, int dtype, bool vec, const Args& A, hipStream_t st) {
    if (dtype == VQA_F32) return by_states<float>(bwd, vec, A, st);
    if (dtype == VQA_BF16) return by_states<bf16>(bwd, vec, A, st);
    return by_states<_Float16>(bwd, vec, A, st);
}

}  // namespace

extern "C" int vqa_scan_ws_bytes(int dtype, int B, int L, int D, int N, int G, long* sizes) {
    if (bad_shape(dtype, B, L, D, N, G) || !sizes) return VQA_ERR_ARG;
    Args A = {};
    A.B = B; A.L = L; A.D = D; A.N = N; A.G = G;
    plan(A, false);
    sizes[0] = 4 * seg_floats(A);
    plan(A, true);
    sizes[1] = 4L * B * kept_tiles(L) * G * A.per_pad * np_of(N);
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
    A.a = a; A.skip = skip; A.dt_bias = dt_bias; A.state = state; A.lengths = lengths;
    A.flags = (softplus ? SOFTPLUS : 0) | (skip ? SKIP : 0);
    A.B = B; A.L = L; A.D = D; A.N = N; A.G = G; A.y = y; A.last = last; A.keep = keep;
    plan(A, false);
    if ((A.segs > 1 && !ws) || !aligned16(ws) || !aligned16(keep) || far_rows(A)) return VQA_ERR_ARG;
    A.seg_h = ws;
    A.seg_dt = ws ? seg_dt_of(A, ws) : nullptr;
    const int e = vqa_elem_bytes(dtype);
    const bool vec = A.per % (16 / e) == 0 && rows_vec(A.x, e) && rows_vec(A.dt, e) && rows_vec(A.gate, e) && on4(y, D, e);
    return by_type(false, dtype, vec, A, static_cast<hipStream_t>(stream));
}

extern "C" int vqa_scan_bwd(void* stream, int dtype, const void* dy, long dy_batch, long dy_row, const float* dlast,
                            const void* x, long x_batch, long x_row, const void* dt, long dt_batch, long dt_row,
                            const void* gate, long gate_batch, long gate_row, const float* a, const void* b, long b_batch,
                            long b_row, const void* c, long c_batch, long c_row, const float* skip, const float* dt_bias,
                            int softplus, const float* state, const int* lengths, int B, int L, int D, int N, int G,
                            const float* keep, void* dx, void* ddt, void* dgate, float* da, void* db, void* dc, float* dskip,
                            float* ddt_bias, float* dstate, float* ws) {
    if (bad_shape(dtype, B, L, D, N, G) || !dy || !x || !dt || !a || !b || !c || (!keep && L > TT) || !dx || !ddt || !da || !db ||
        !dc || !ws || (gate && !dgate) || !aligned16(ws) || !aligned16(keep))
        return VQA_ERR_ARG;
    Args A = {};
    A.dy = {dy, dy_batch, dy_row};
    A.x = {x, x_batch, x_row}; A.dt = {dt, dt_batch, dt_row}; A.gate = {gate, gate_batch, gate_row};
    A.b = {b, b_batch, b_row}; A.c = {c, c_batch, c_row};
    A.a = a; A.skip = skip; A.dt_bias = dt_bias; A.dlast = dlast; A.state = state; A.lengths = lengths;
    A.flags = (softplus ? SOFTPLUS : 0) | (skip ? SKIP : 0);
    A.B = B; A.L = L; A.D = D; A.N = N; A.G = G; A.keep = const_cast<float*>(keep);
    A.dx = dx; A.ddt = ddt; A.dgate = dgate; A.dstate = dstate;
    if (far_rows(A)) return VQA_ERR_ARG;
    plan(A, true);
    A.seg_h = ws;
    A.seg_dt = seg_dt_of(A, ws);
    A.part_p = ws + seg_floats(A);
    A.part_bc = A.part_p + part_p_floats(A);
    A.params = (int)(((long)G * A.per_pad * (np_of(N) + 2) + 63) / 64);
    A.da = da; A.db = db; A.dc = dc; A.dskip = dskip; A.dbias = ddt_bias;
    const int e = vqa_elem_bytes(dtype);
    const bool vec = A.per % (16 / e) == 0 && rows_vec(A.x, e) && rows_vec(A.dt, e) && rows_vec(A.gate, e) &&
                     rows_vec(A.dy, e) && on4(dx, D, e) && on4(ddt, D, e) && on4(dgate, D, e);
    return by_type(true, dtype, vec, A, static_cast<hipStream_t>(stream));
}

namespace {
template <typename T>
int token(hipStream_t st, const Rows& x, float* state, long sb, const Rows& dt, const Rows& gate, const Rows& b, const Rows& c,
          const float* a, const float* skip, const float* bias, int softplus, int B, int D, int N, int G, void* y) {
    constexpr int e = sizeof(T);
    const bool vec = N % 4 == 0 && sb % 4 == 0 && aligned16(state) && aligned16(a) && vqa_vec_ok(b.p, b.batch, e, 4 * e) &&
                     vqa_vec_ok(c.p, c.batch, e, 4 * e);
    const int ln = N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16, blocks = (D * ln + 255) / 256;
#define VQA_TOKEN(LN)                                                                                                    \
    if (ln == LN) {                                                                                                      \
        if (vec) scan_token<T, LN, true><<<(unsigned)(B * blocks), 256, 0, st>>>(x, state, sb, dt, gate, b, c, a, skip, bias, softplus, D, N, D / G, blocks, static_cast<T*>(y)); \
        else scan_token<T, LN, false><<<(unsigned)(B * blocks), 256, 0, st>>>(x, state, sb, dt, gate, b, c, a, skip, bias, softplus, D, N, D / G, blocks, static_cast<T*>(y));    \
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
    // (at most 16 lanes a channel, 256 threads a workgroup, and a grid has fewer than 2^32 threads)
    if (bad_shape(dtype, B, 1, D, N, G) || (double)B * ((D + 15) / 16) > 1.6e7 || !x || !state || !dt || !a || !b || !c || !y) return VQA_ERR_ARG;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const Rows rx = {x, x_batch, 0}, rd = {dt, dt_batch, 0}, rg = {gate, gate_batch, 0}, rb = {b, b_batch, 0}, rc = {c, c_batch, 0};
    if (dtype == VQA_F32) return token<float>(st, rx, state, state_batch, rd, rg, rb, rc, a, skip, dt_bias, softplus, B, D, N, G, y);
    if (dtype == VQA_BF16) return token<bf16>(st, rx, state, state_batch, rd, rg, rb, rc, a, skip, dt_bias, softplus, B, D, N, G, y);
    return token<_Float16>(st, rx, state, state_batch, rd, rg, rb, rc, a, skip, dt_bias, softplus, B, D, N, G, y);
}
