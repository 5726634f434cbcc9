// Rotary positions in general, and the append of new tokens to a paged cache with them (gfx950), f32.
//
// A head's first `rot` columns are pairs (i, i + rot / 2), or (2 i, 2 i + 1); pair i of a row at position p is turned
// by the angle p f_i, and lengthened by the amplitude a:
//     (lo, hi) -> a (lo cos - hi sin, hi cos + lo sin);     back: a (lo cos + hi sin, hi cos - lo sin),
// the transpose, which is what gradients go through.  The other columns are copied.  Positions come from memory, one
// a row, frequencies with the arguments.  Angle, cosine, sine and the products are in 64 bits, with one rounding
// to f32 at the end: at position 10^5 an f32 angle would be off by 4e-3.
//
// A workgroup takes a row, whose angles its threads compute before they share them for every head of q and k, or one of
// a.slices parts of the row's heads: few rows are cut into parts for more workgroups.  A thread then takes VW pairs of a
// head at a time, 16 bytes a load where widths allow, several such units in flight.  Bound: HBM: 8192 rows of 32 + 8
// heads at d = 128 61 to 63 us, 5.4 TB/s (a copy of 2 GiB 5.0).  Measured on MI355X (us): with two rows to a workgroup 64,
// with four 70; a quarter of each head turned 59.6, with 16 rows to a workgroup (16 angles each) 122; the new tokens of 48
// sequences, 1936 of 16 + 4 heads at d = 256, and their masks, 23.5 with two units in flight, 31 with four.
//
// The append beside zt_rope_paged_*, which turns whole heads, halves as pairs, at positions that the host counts up, with
// zt_rope_forward's angles bit for bit, and several tokens to a workgroup where heads are narrow.  On the device (us, that one
// / this one): 64 tokens, one a sequence, of 32 + 8 heads at d = 128 8.0 / 5.4, 1920 of 16 + 4 at d = 256 23.8 / 23.8, 8000 of
// 32 + 8 at d = 128 68.6 / 68.0, 8000 of 4 + 2 at d = 32 10.6 / 15.9.
#include "common.h"
#include "args.h"
#include "paged.h"

template <int N>
struct Vec {
    typedef float type __attribute__((ext_vector_type(N)));
};

// A row's angles into LDS.
DEVI void turn_angles(const TurnArgs &a, int t, double2 *tab) {
    for (int i = threadIdx.x; i < a.rot >> 1; i += 256) {
        double s, c;
        sincos((double)a.pos[t] * a.freq[i], &s, &c);
        tab[i] = double2{c * a.amplitude, s * a.sine};
    }
}

// Unit u of a head: VW pairs, or, past its pairs, as many columns as a load takes.  Read from x, written to y, both at
// the head's first column; tab: the row's angles.
template <int VW, bool INTER>
struct TurnUnit {
    static constexpr int N = VW == 1 || INTER ? 2 * VW : VW;  // columns of a copy
    typedef typename Vec<VW == 1 ? 2 : VW>::type vec;
    typedef typename Vec<N>::type copy;
    float in[2][VW];
    int at;  // its first column, of a turn the first pair
    bool turns;

    DEVI void read(const TurnArgs &a, int u, const float *x) {
        const int half = a.rot >> 1, pairs = half / VW;
        turns = u < pairs;
        at = turns ? u * VW : a.rot + (u - pairs) * N;
        if constexpr (INTER) {
            const copy z = __builtin_nontemporal_load(reinterpret_cast<const copy *>(x + (turns ? 2 * at : at)));
#pragma unroll
            for (int e = 0; e < VW; ++e) {
                in[0][e] = z[2 * e];
                in[1][e] = z[2 * e + 1];
            }
        } else if constexpr (VW == 1) {
            in[0][0] = x[at];
            in[1][0] = x[at + (turns ? half : 1)];
        } else {
            const vec lo = __builtin_nontemporal_load(reinterpret_cast<const vec *>(x + at));
            vec hi = lo;
            if (turns) hi = __builtin_nontemporal_load(reinterpret_cast<const vec *>(x + at + half));
#pragma unroll
            for (int e = 0; e < VW; ++e) {
                in[0][e] = lo[e];
                in[1][e] = hi[e];
            }
        }
    }
    DEVI void write(const TurnArgs &a, const double2 *tab, float *y) {
        const int half = a.rot >> 1;
        if (turns) {
#pragma unroll
            for (int e = 0; e < VW; ++e) {
                const double2 cs = tab[at + e];
                const double lo = in[0][e], hi = in[1][e];
                in[0][e] = (float)(lo * cs.x - hi * cs.y);
                in[1][e] = (float)(hi * cs.x + lo * cs.y);
            }
        }
        if constexpr (INTER) {
            copy z;
#pragma unroll
            for (int e = 0; e < VW; ++e) {
                z[2 * e] = in[0][e];
                z[2 * e + 1] = in[1][e];
            }
            *reinterpret_cast<copy *>(y + (turns ? 2 * at : at)) = z;
        } else if constexpr (VW == 1) {
            y[at] = in[0][0];
            y[at + (turns ? half : 1)] = in[1][0];
        } else {
            vec lo, hi;
#pragma unroll
            for (int e = 0; e < VW; ++e) {
                lo[e] = in[0][e];
                hi[e] = in[1][e];
            }
            *reinterpret_cast<vec *>(y + at) = lo;
            if (turns) *reinterpret_cast<vec *>(y + at + half) = hi;
        }
    }
};

// Units of a head; in place its pairs alone.
template <int VW, bool INTER>
DEVI int turn_units(const TurnArgs &a, bool in_place) {
    return (a.rot >> 1) / VW + (in_place ? 0 : (a.dim - a.rot) / (VW == 1 || INTER ? 2 * VW : VW));
}

template <int VW, bool INTER>
DEVI void turn_rows(const TurnArgs &a) {
    constexpr int U = 4;  // units in flight
    __shared__ double2 tab[ZT_MAX_DIM / 2];
    const int slice = (int)blockIdx.x % a.slices;
    const size_t t = (size_t)a.row0 + blockIdx.x / a.slices;
    const int units = turn_units<VW, INTER>(a, a.q == a.q_out && a.k == a.k_out), tasks = (a.H + a.Hkv) * units;
    const int per_slice = (tasks + a.slices - 1) / a.slices;
    const int j0 = slice * per_slice, j1 = min(tasks, j0 + per_slice);
    const size_t q0 = t * a.H * a.dim, k0 = t * a.Hkv * a.dim;
    const float *const q = a.q + q0, *const k = a.k + k0;
    float *const q_out = a.q_out + q0, *const k_out = a.k_out + k0;
    turn_angles(a, (int)t, tab);
    __syncthreads();
    for (int j = j0 + (int)threadIdx.x; j < j1; j += 256 * U) {
        TurnUnit<VW, INTER> x[U];
        float *y[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int e = j + 256 * i;
            if (e >= j1) break;
            const int h = e / units, at = (h < a.H ? h : h - a.H) * a.dim;
            x[i].read(a, e - h * units, (h < a.H ? q : k) + at);
            y[i] = (h < a.H ? q_out : k_out) + at;
        }
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (j + 256 * i < j1) x[i].write(a, tab, y[i]);
    }
}

// New tokens of a ragged batch: q and k turned, k and v written to the tokens' rows of the cache, those rows'
// accumulated weights cleared.  A row whose page is none of the pool's is not written.
template <int VW, bool INTER>
DEVI void turn_paged(const TurnPagedArgs &p) {
    constexpr int U = 2;  // units in flight
    const TurnArgs &a = p.turn;
    typedef TurnUnit<VW, INTER> Unit;
    __shared__ double2 tab[ZT_MAX_DIM / 2];
    const int slice = (int)blockIdx.x % a.slices, tok = a.row0 + (int)(blockIdx.x / a.slices);
    const int lane = lane_id(), b0 = p.b[lane], f0 = p.first[lane], s0 = lane < p.ns ? p.q0[lane] : INT32_MAX;
    // The token's sequence, the last that does not begin past it, and its row there and in the pool.
    const int sq = __builtin_amdgcn_readfirstlane(__popcll(__builtin_amdgcn_ballot_w64(s0 <= tok)) - 1);
    const int b = __builtin_amdgcn_readlane(b0, sq);
    const int at = __builtin_amdgcn_readlane(f0, sq) + tok - __builtin_amdgcn_readlane(s0, sq);
    const int row = pool_row(p.pool, p.pool.table + (size_t)b * p.pool.table_stride, at);
    turn_angles(a, tok, tab);
    __syncthreads();
    const size_t t = (size_t)tok, q0 = t * a.H * a.dim, k0 = t * a.Hkv * a.dim;
    const float *const q = a.q + q0, *const k = a.k + k0, *const v = p.v_new + k0;
    float *const q_out = a.q_out + q0;
    float *const k_out = p.pool.k + (size_t)row * a.Hkv * a.dim, *const v_out = p.pool.v + (size_t)row * a.Hkv * a.dim;
    // The token's tasks: its turns, q's heads (if any) then k's, and the copies of v, in vectors as its units'.
    const int uq = turn_units<VW, INTER>(a, a.q == a.q_out), uk = turn_units<VW, INTER>(a, false);
    const int nq = (a.q ? a.H : 0) * uq, nk = a.Hkv * uk;
    const int tasks = row < 0 ? nq : nq + nk + a.Hkv * a.dim / Unit::N;
    const int per_slice = (tasks + a.slices - 1) / a.slices;
    const int j0 = slice * per_slice, j1 = min(tasks, j0 + per_slice);
    for (int j = j0 + (int)threadIdx.x; j < j1; j += 256 * U) {
        Unit x[U];
        typename Unit::copy c[U];
        float *y[U];
        bool turn[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int e = j + 256 * i;
            y[i] = nullptr;
            if (e >= j1) break;
            turn[i] = e < nq + nk;
            if (turn[i]) {
                const bool is_q = e < nq;
                const int of = is_q ? e : e - nq, units = is_q ? uq : uk, h = of / units;
                x[i].read(a, of - h * units, (is_q ? q : k) + h * a.dim);
                y[i] = (is_q ? q_out : k_out) + h * a.dim;
            } else {
                const int col = Unit::N * (e - nq - nk);
                c[i] = __builtin_nontemporal_load(reinterpret_cast<const typename Unit::copy *>(v + col));
                y[i] = v_out + col;
            }
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (j + 256 * i >= j1) break;
            if (turn[i]) x[i].write(a, tab, y[i]);
            else *reinterpret_cast<typename Unit::copy *>(y[i]) = c[i];
        }
    }
    if (p.w && slice == 0)
        for (int h = threadIdx.x; h < a.Hkv; h += 256) p.w[((size_t)b * a.Hkv + h) * p.w_stride + at] = 0.f;
}

#define ZT_TURN(NAME, VW, INTER)                                                                    \
    extern "C" __global__ void __launch_bounds__(256) zt_turn_##NAME(TurnArgs a) { turn_rows<VW, INTER>(a); } \
    extern "C" __global__ void __launch_bounds__(256) zt_turn_paged_##NAME(TurnPagedArgs a) { turn_paged<VW, INTER>(a); }
ZT_TURN(half4, 4, false)
ZT_TURN(half2, 2, false)
ZT_TURN(half1, 1, false)
ZT_TURN(inter2, 2, true)
ZT_TURN(inter1, 1, true)
