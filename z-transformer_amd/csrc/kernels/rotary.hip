// Rotary positions in general, and the append of new tokens to a paged cache with them (gfx950), f32.
//
// A head's first `rot` columns are pairs (i, i + rot / 2), or (2 i, 2 i + 1); pair i of a row at position p is turned
// by the angle p f_i, and lengthened by the amplitude a:
//     (lo, hi) -> a (lo cos - hi sin, hi cos + lo sin);     back: a (lo cos + hi sin, hi cos - lo sin),
// the transpose, which is what gradients go through.  The other columns are copied.  Positions come from memory, one
// a row, frequencies with the arguments.  Angle, cosine, sine and the products are in 64 bits, with one rounding
// to f32 at the end: at position 10^5 an f32 angle would be off by 4e-3.
//
// A workgroup takes a group of rows, so that its threads compute one (row, pair) angle each, before they share them
// for every head of q and k, and one of a.slices parts of the rows' heads: few rows are cut into parts for more
// workgroups.  A thread then takes VW pairs of a head at a time, 16 bytes a load where widths allow.  Bound: HBM.
#include "common.h"
#include "args.h"
#include "paged.h"

constexpr int kTurnRows = 16;  // rows of a workgroup at most

template <int N>
struct Vec {
    typedef float type __attribute__((ext_vector_type(N)));
};

// Angles of rows t0 .. t0 + nt - 1 into LDS.
DEVI void turn_angles(const TurnArgs &a, int t0, int nt, double2 *tab) {
    const int half = a.rot >> 1;
    for (int j = threadIdx.x; j < nt * half; j += 256) {
        const int tl = j / half, i = j - tl * half;
        double s, c;
        sincos((double)a.pos[t0 + tl] * a.freq[i], &s, &c);
        tab[j] = double2{c * a.amplitude, s * a.sine};
    }
}

// Unit u of a head (VW pairs, or, past its pairs, as many columns as a load takes) from x to y, both at the head's
// first column; tab: the row's angles.
template <int VW, bool INTER>
DEVI void turn_unit(const TurnArgs &a, const double2 *tab, int u, const float *x, float *y) {
    constexpr int N = VW == 1 || INTER ? 2 * VW : VW;  // columns of a copy
    typedef typename Vec<VW == 1 ? 2 : VW>::type vec;
    typedef typename Vec<N>::type copy;
    const int half = a.rot >> 1, pairs = half / VW;
    if (u >= pairs) {
        const int c = a.rot + (u - pairs) * N;
        *reinterpret_cast<copy *>(y + c) = __builtin_nontemporal_load(reinterpret_cast<const copy *>(x + c));
        return;
    }
    float in[2][VW], out[2][VW];
    const int i = u * VW;
    if constexpr (INTER) {
        const copy z = __builtin_nontemporal_load(reinterpret_cast<const copy *>(x + 2 * i));
#pragma unroll
        for (int e = 0; e < VW; ++e) {
            in[0][e] = z[2 * e];
            in[1][e] = z[2 * e + 1];
        }
    } else if constexpr (VW == 1) {
        in[0][0] = x[i];
        in[1][0] = x[i + half];
    } else {
        const vec lo = __builtin_nontemporal_load(reinterpret_cast<const vec *>(x + i));
        const vec hi = __builtin_nontemporal_load(reinterpret_cast<const vec *>(x + i + half));
#pragma unroll
        for (int e = 0; e < VW; ++e) {
            in[0][e] = lo[e];
            in[1][e] = hi[e];
        }
    }
#pragma unroll
    for (int e = 0; e < VW; ++e) {
        const double2 cs = tab[i + e];
        const double lo = in[0][e], hi = in[1][e];
        out[0][e] = (float)(lo * cs.x - hi * cs.y);
        out[1][e] = (float)(hi * cs.x + lo * cs.y);
    }
    if constexpr (INTER) {
        copy z;
#pragma unroll
        for (int e = 0; e < VW; ++e) {
            z[2 * e] = out[0][e];
            z[2 * e + 1] = out[1][e];
        }
        *reinterpret_cast<copy *>(y + 2 * i) = z;
    } else if constexpr (VW == 1) {
        y[i] = out[0][0];
        y[i + half] = out[1][0];
    } else {
        vec lo, hi;
#pragma unroll
        for (int e = 0; e < VW; ++e) {
            lo[e] = out[0][e];
            hi[e] = out[1][e];
        }
        *reinterpret_cast<vec *>(y + i) = lo;
        *reinterpret_cast<vec *>(y + i + half) = hi;
    }
}

// Units of a head; in place its pairs alone.
template <int VW, bool INTER>
DEVI int turn_units(const TurnArgs &a, bool in_place) {
    return (a.rot >> 1) / VW + (in_place ? 0 : (a.dim - a.rot) / (VW == 1 || INTER ? 2 * VW : VW));
}

template <int VW, bool INTER>
DEVI void turn_rows(const TurnArgs &a) {
    __shared__ double2 tab[256];
    const int half = a.rot >> 1, per = min(kTurnRows, 256 / half);
    const int group = (int)blockIdx.x / a.slices, slice = (int)blockIdx.x % a.slices;
    const int t0 = a.row0 + group * per, nt = min(per, a.row0 + a.rows - t0);
    turn_angles(a, t0, nt, tab);
    __syncthreads();
    const int units = turn_units<VW, INTER>(a, a.q == a.q_out && a.k == a.k_out), tasks = (a.H + a.Hkv) * units;
    const int per_slice = (tasks + a.slices - 1) / a.slices;
    const int j0 = slice * per_slice, nj = min(per_slice, tasks - j0);
    const size_t qld = (size_t)a.H * a.dim, kld = (size_t)a.Hkv * a.dim;
    const float *const q = a.q, *const k = a.k;
    float *const q_out = a.q_out, *const k_out = a.k_out;
    for (int e = threadIdx.x; e < nt * nj; e += 256) {
        const int tl = e / nj, j = j0 + e - tl * nj, h = j / units, u = j - h * units;
        const size_t t = (size_t)(t0 + tl);
        const bool is_q = h < a.H;
        const size_t at = is_q ? t * qld + (size_t)h * a.dim : t * kld + (size_t)(h - a.H) * a.dim;
        turn_unit<VW, INTER>(a, tab + tl * half, u, (is_q ? q : k) + at, (is_q ? q_out : k_out) + at);
    }
}

// New tokens of a ragged batch: q and k turned, k and v written to the tokens' rows of the cache, those rows'
// accumulated weights cleared.  A row whose page is none of the pool's is not written.
template <int VW, bool INTER>
DEVI void turn_paged(const TurnPagedArgs &p) {
    const TurnArgs &a = p.turn;
    constexpr int VV = VW == 1 || INTER ? 2 * VW : VW;  // of v's copies
    typedef typename Vec<VV>::type vvec;
    __shared__ double2 tab[256];
    __shared__ int row_of[kTurnRows], seq_of[kTurnRows], at_of[kTurnRows];
    const int half = a.rot >> 1, per = min(kTurnRows, 256 / half);
    const int group = (int)blockIdx.x / a.slices, slice = (int)blockIdx.x % a.slices;
    const int t0 = a.row0 + group * per, nt = min(per, a.row0 + a.rows - t0);
    if (threadIdx.x < 64) {  // a wave finds the tokens' rows
        const int lane = threadIdx.x, q0 = p.q0[lane], b = p.b[lane], row0 = p.first[lane];
        const int t = t0 + min(lane, nt - 1);
        int sq = 0;  // the last sequence that does not begin past the token
        for (int s = 1; s < p.ns; ++s) sq = __builtin_amdgcn_readlane(q0, s) <= t ? s : sq;
        const int at = __shfl(row0, sq, 64) + t - __shfl(q0, sq, 64), bs = __shfl(b, sq, 64);
        if (lane < nt) {
            row_of[lane] = pool_row(p.pool, p.pool.table + (size_t)bs * p.pool.table_stride, at);
            seq_of[lane] = bs;
            at_of[lane] = at;
        }
    }
    turn_angles(a, t0, nt, tab);
    __syncthreads();
    const size_t qld = (size_t)a.H * a.dim, kld = (size_t)a.Hkv * a.dim;
    // A token's tasks: its turns, q's heads (if any) then k's, and the copies of v.
    const int uq = turn_units<VW, INTER>(a, a.q == a.q_out), uk = turn_units<VW, INTER>(a, false);
    const int nq = (a.q ? a.H : 0) * uq, nk = a.Hkv * uk;
    const int tasks = nq + nk + (int)(kld / VV);
    const int per_slice = (tasks + a.slices - 1) / a.slices;
    const int j0 = slice * per_slice, nj = min(per_slice, tasks - j0);
    for (int e = threadIdx.x; e < nt * nj; e += 256) {
        const int tl = e / nj, j = j0 + e - tl * nj;
        const size_t t = (size_t)(t0 + tl);
        const int row = row_of[tl];
        if (j < nq) {
            const int h = j / uq;
            const size_t at = t * qld + (size_t)h * a.dim;
            turn_unit<VW, INTER>(a, tab + tl * half, j - h * uq, a.q + at, a.q_out + at);
        } else if (row >= 0 && j < nq + nk) {
            const int h = (j - nq) / uk;
            turn_unit<VW, INTER>(a, tab + tl * half, j - nq - h * uk, a.k + t * kld + (size_t)h * a.dim,
                                 p.pool.k + (size_t)row * kld + (size_t)h * a.dim);
        } else if (row >= 0) {
            const size_t col = (size_t)VV * (j - nq - nk);
            *reinterpret_cast<vvec *>(p.pool.v + (size_t)row * kld + col) =
                __builtin_nontemporal_load(reinterpret_cast<const vvec *>(p.v_new + t * kld + col));
        }
    }
    if (p.w && slice == 0)
        for (int e = threadIdx.x; e < nt * a.Hkv; e += 256) {
            const int tl = e / a.Hkv, h = e - tl * a.Hkv;
            p.w[((size_t)seq_of[tl] * a.Hkv + h) * p.w_stride + at_of[tl]] = 0.f;
        }
}

#define ZT_TURN(NAME, VW, INTER)                                                                    \
    extern "C" __global__ void __launch_bounds__(256) zt_turn_##NAME(TurnArgs a) { turn_rows<VW, INTER>(a); } \
    extern "C" __global__ void __launch_bounds__(256) zt_turn_paged_##NAME(TurnPagedArgs a) { turn_paged<VW, INTER>(a); }
ZT_TURN(half4, 4, false)
ZT_TURN(half2, 2, false)
ZT_TURN(half1, 1, false)
ZT_TURN(inter2, 2, true)
ZT_TURN(inter1, 1, true)
