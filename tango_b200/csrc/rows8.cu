// 8-bit rows: packing, unpacking, and activations whose saved input is held in them.
//
//   pack     : s = max|x| / 127 over a group, codes x / s exactly rounded; with an activation also y = f(x) in the same pass
//   unpack   : code * s
//   backward : dx = dy * f'(code * s), from the 8-bit copy alone
//
// Bound by HBM in principle: pack 5 bytes an fp32 element (4 read, 1 written), unpack 5, activation forward 9, backward 9.  A group
// is owned by a few lanes, each with R times four neighbouring elements LPG * 4 apart (a load and the store of four codes are
// contiguous over the lanes), so that x is read once and stays in registers.  Measured, GB/s of those bytes:
//   contiguous groups of 4, 8, .. 128 columns: GELU of 232965 x 256 forward 98 us (5.5 TB/s), backward 79 (6.8, dy partly in L2);
//     three matrices of 29.8 M elements, one launch, 94 us (4.8): 26 instructions an element keep the issue slots three quarters busy
//   602 columns, fp32: pack 151 us (4.7: 28 instructions an element, issue slots 76 % busy), unpack 110 (6.4); pairs of elements, half a
//     sector, 217 and 163
//   601 columns, bf16, SiLU: forward 176 us (2.9), backward 146 (3.5): 49 and 39 instructions an element, issue slots 81 and 78 % busy
// An earlier form with four elements a lane and 32 lanes a group took 408, 215 and 406 us where the first of each pair stands.
#include "rows8.cuh"

#include <initializer_list>

namespace tango {

constexpr int kBlock = 256;
constexpr int kMaxGroup = 1024, kMaxJobs = 4;
enum { ACT_NONE = -1, ACT_ELU = 0, ACT_GELU = 1, ACT_SILU = 2 };

struct Rows8Args {
    const void *x[kMaxJobs];      // pack: input; backward: gradient dy
    int64_t ldx[kMaxJobs];
    int8_t *q[kMaxJobs];
    float *scale[kMaxJobs];       // [rows, groups], of group i at i * scale_stride
    int64_t scale_stride[kMaxJobs];
    int run[kMaxJobs];            // 0, or the codes of a run of an interleaved matrix
    void *y;                      // activation forward: y; unpack and backward: output
    int64_t ldy;
    int64_t rows, cols, items;    // items = rows * groups
    int32_t group, groups, pitch; // bytes between the codes of two groups
    int32_t tile;                 // codes that the lanes of a group have to cover
    int64_t ldq;
    FastDiv by_groups;
    int wide;                     // 2^31 groups or more
    int jobs;                     // matrices: blocks take them in turn, so that the runs of interleaved ones meet in L2
    int mode, act;
    int over;                     // input and output lie differently on the boundaries of four elements
    uint64_t seed, call;
    const unsigned long long *step;
};

template <int K> struct Kind { static constexpr int value = K; };

__device__ __forceinline__ float exp_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
    return y;
}
// x / y for y >= 1
__device__ __forceinline__ float over(float x, float y) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
    return x * r;
}
// Upper tail of the normal distribution at |x| times two, erfc(|x| / sqrt(2)), with e = exp(-x^2 / 2): the rational formula 7.1.26
// of Abramowitz and Stegun's handbook (|error| < 1.5e-7), which shares the exponential with the density.  The error is of the
// size of fp32's rounding of 1 + erf, but a choice all the same: GELU of 232965 x 256 normal numbers (1.5 wide) and its gradient are
// 9.5e-8 of their norm from 64 bits, erf and exp in full 4.9e-8; for x below about -5, where 1 + erf cancels, the formula is closer.
__device__ __forceinline__ float normal_tails(float x, float e) {
    const float t = over(1.f, fmaf(0.3275911f * 0.70710678118654752f, fabsf(x), 1.f));
    float p = fmaf(1.061405429f, t, -1.453152027f);
    p = fmaf(p, t, 1.421413741f);
    p = fmaf(p, t, -0.284496736f);
    p = fmaf(p, t, 0.254829592f);
    return p * t * e;
}
template <int act>
__device__ __forceinline__ float activate(float x) {
    if (act == ACT_ELU) return x > 0.f ? x : expm1f(x);
    if (act == ACT_GELU) {
        const float half = 0.5f * normal_tails(x, exp_fast(-0.5f * x * x));
        return x * (x > 0.f ? 1.f - half : half);
    }
    return over(x, 1.f + exp_fast(-x));
}
// The slope is taken at the 8-bit copy, off by at most half a step; each f is smooth enough (|f''| <= 1, one-sided at ELU's 0,
// where the slope is continuous) that the slope moves by no more than that.
template <int act>
__device__ __forceinline__ float slope_of(float t) {
    if (act == ACT_ELU) return t > 0.f ? 1.f : exp_fast(t);
    if (act == ACT_GELU) {
        const float e = exp_fast(-0.5f * t * t), half = 0.5f * normal_tails(t, e);
        // behind 2^64 the density is 0 and t may be too large to multiply by it
        return fmaf(fabsf(t) < 1e19f ? t * 0.39894228040143268f : 0.f, e, t > 0.f ? 1.f - half : half);
    }
    const float s = over(1.f, 1.f + exp_fast(-t));
    return s == 0.f ? 0.f : s * fmaf(t, 1.f - s, 1.f);
}

// f with the activation as a constant: one branch for all elements of a thread.
template <class F>
__device__ __forceinline__ void with_act(int act, F f) {
    if (act == ACT_ELU) f(Kind<ACT_ELU>{});
    else if (act == ACT_GELU) f(Kind<ACT_GELU>{});
    else f(Kind<ACT_SILU>{});
}

// Where item `i` (a group of a row) lies.
struct Where {
    int64_t row, x;    // row, and the item's first element in a matrix of leading dimension ld
    int32_t g, n;      // group, its elements
};
__device__ __forceinline__ Where locate(const Rows8Args &a, int64_t i, int64_t ld) {
    Where w;
    if (a.wide) {
        w.row = i / a.groups;
        w.g = (int32_t)(i - w.row * a.groups);
        w.x = w.row * ld + (int64_t)w.g * a.group;
        const int64_t left = a.cols - (int64_t)w.g * a.group;
        w.n = left < a.group ? (int32_t)left : a.group;
    } else {           // items, columns and leading dimensions below 2^31
        const uint32_t r = quotient((uint32_t)i, a.by_groups), at = ((uint32_t)i - r * (uint32_t)a.groups) * (uint32_t)a.group;
        w.row = r;
        w.g = (int32_t)((uint32_t)i - r * (uint32_t)a.groups);
        w.x = (int64_t)((uint64_t)r * (uint32_t)ld + at);
        w.n = min((int32_t)((uint32_t)a.cols - at), a.group);
    }
    return w;
}
// First byte of an item's codes (of a plain matrix), and its bytes with the zeros behind them.
__device__ __forceinline__ int64_t code_place(const Rows8Args &a, const Where &w) { return w.row * a.ldq + (int64_t)w.g * a.pitch; }
__device__ __forceinline__ int code_width(const Rows8Args &a, const Where &w) {
    return w.g == a.groups - 1 ? (int)(a.ldq - (int64_t)w.g * a.pitch) : a.pitch;
}

// LPG lanes a group, R times four elements a lane, U groups in flight.
template <int LPG, int R> struct Tile {
    static constexpr int U = R == 1 ? 4 : R == 2 ? 2 : 1;
    static constexpr int kGroups = kBlock / LPG;        // groups a block works on at a time
    static constexpr int kItems = kGroups * U;
    static constexpr int kElements = kItems * LPG * R * 4;
};

// How the elements are reached: in the aligned pieces of four that hold them (rows of any pitch), four at a time, or in one run.
enum { TURNED = 0, WIDE = 4, FLAT = 8 };

// ---- a lane's elements of a group: slots of four neighbours at lane * 4, (lane + LPG) * 4, ..
// In rows of any pitch a group starts `skip` elements behind a boundary of 16 (8) bytes, and slot k takes the aligned piece k: the
// elements 4 k - skip + i.  The `skip` places that this leaves free in slot 0 take the last elements of a full group, which lie in
// a piece of their own, so that the group is turned by `skip` within its slots and fills as many as before.  Loads, the maximum,
// the activation and stores do not mind; only the codes are turned back, in one exchange of words.  169343 x 601 bf16, SiLU,
// forward: 174 us; with the elements shifted into place 216, with single accesses 373.
template <int LPG, int R> constexpr int kSlots = LPG * R * 4;
template <class T, int ACCESS> __device__ __forceinline__ int skip_of(const T *p) {
    return ACCESS == TURNED ? (int)(reinterpret_cast<uintptr_t>(p) / sizeof(T) & 3) : 0;
}
// Element in place i of slot k.
template <int LPG, int R> __device__ __forceinline__ int element(int k, int i, int skip) {
    const int e = k * 4 - skip + i;
    return e < 0 ? e + kSlots<LPG, R> : e;
}
__device__ __forceinline__ void load_piece(const float *p, float *v) {
    const float4 t = __ldg(reinterpret_cast<const float4 *>(p));
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
}
template <class T> __device__ __forceinline__ void load_piece(const T *p, float *v) {
    const uint2 t = __ldg(reinterpret_cast<const uint2 *>(p));
    unpack2<T>(t.x, v[0], v[1]);
    unpack2<T>(t.y, v[2], v[3]);
}
__device__ __forceinline__ void store_piece(float *p, const float *v) { *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]); }
template <class T> __device__ __forceinline__ void store_piece(T *p, const float *v) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
}

// n elements at p; [begin, end): the matrix, outside of which nothing is read.
template <class T, int ACCESS, int LPG, int R>
__device__ __forceinline__ void load_group(const T *p, int n, const T *begin, const T *end, float (&v)[R * 4]) {
    const int lane = threadIdx.x % LPG;
    if constexpr (ACCESS == WIDE) {
#pragma unroll
        for (int r = 0; r < R; ++r) load4<T, WIDE>(p + (lane + r * LPG) * 4, n - (lane + r * LPG) * 4, v + 4 * r);
    } else {
        const int skip = skip_of<T, ACCESS>(p), pieces = n > 0 ? (n + skip + 3) / 4 : 0;
        const T *first = p - skip;
#pragma unroll
        for (int k = 0; k < R * 4; ++k) v[k] = 0.f;
        if (first >= begin && first + pieces * 4 <= end) {
            float last[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (lane + r * LPG < pieces) load_piece(first + (lane + r * LPG) * 4, v + 4 * r);
            if (lane == 0 && LPG * R < pieces) load_piece(first + kSlots<LPG, R>, last);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int left = n + skip - (lane + r * LPG) * 4;
                if (r == 0 && lane == 0) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = element<LPG, R>(0, i, skip) < n ? (i < skip ? last[i] : v[i]) : 0.f;
                } else if (left < 4) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[4 * r + i] = i < left ? v[4 * r + i] : 0.f;
                }
            }
        } else {                        // the matrix begins or ends inside a piece
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = element<LPG, R>(lane + r * LPG, i, skip);
                    if (e < n) v[4 * r + i] = to_float(p[e]);
                }
        }
    }
}
template <class T, int ACCESS, int LPG, int R>
__device__ __forceinline__ void store_group(T *p, int n, const float (&v)[R * 4]) {
    const int lane = threadIdx.x % LPG;
    if constexpr (ACCESS == WIDE) {
#pragma unroll
        for (int r = 0; r < R; ++r) store4<T, WIDE>(p + (lane + r * LPG) * 4, n - (lane + r * LPG) * 4, v + 4 * r);
    } else {
        const int skip = skip_of<T, ACCESS>(p);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int e = (lane + r * LPG) * 4 - skip;
            if (e >= 0 && e + 4 <= n) {
                store_piece(p + e, v + 4 * r);
            } else if (r == 0 && e < 0) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int at = element<LPG, R>(0, i, skip);
                    if (at < n) from_float(v[i], p[at]);
                }
            } else if (e < n) {
#pragma unroll
                for (int i = 0; i < 3; ++i)
                    if (e + i < n) from_float(v[4 * r + i], p[e + i]);
            }
        }
    }
}
// The lane (of a group's LPG) before or after this one, as a lane of the warp.
template <int LPG> __device__ __forceinline__ int neighbour(int by) {
    return ((threadIdx.x & 31) & ~(LPG - 1)) + ((threadIdx.x + by) & (LPG - 1));
}
// Codes of the slots, turned, to the words of the codes in order, and back.
template <int LPG, int R> __device__ __forceinline__ void turn_back(uint32_t (&word)[R], int skip) {
    const bool wraps = threadIdx.x % LPG == 0;
    uint32_t next[R];
#pragma unroll
    for (int r = 0; r < R; ++r) next[r] = __shfl_sync(0xffffffffu, wraps ? word[(r + 1) % R] : word[r], neighbour<LPG>(1));
#pragma unroll
    for (int r = 0; r < R; ++r) word[r] = __byte_perm(word[r], next[r], 0x3210 + 0x1111 * skip);
}
template <int LPG, int R> __device__ __forceinline__ void turn(uint32_t (&word)[R], int skip) {
    const bool wraps = threadIdx.x % LPG == LPG - 1;
    uint32_t before[R];
#pragma unroll
    for (int r = 0; r < R; ++r) before[r] = __shfl_sync(0xffffffffu, wraps ? word[(r + R - 1) % R] : word[r], neighbour<LPG>(LPG - 1));
#pragma unroll
    for (int r = 0; r < R; ++r) word[r] = __byte_perm(before[r], word[r], 0x7654 - 0x1111 * skip);
}
// Elements turned by `from` to elements turned by `to`, for an output that lies otherwise on its boundaries than the input.
template <int LPG, int R> __device__ __forceinline__ void turn_over(float (&v)[R * 4], int from, int to) {
    const bool first = threadIdx.x % LPG == 0, last = threadIdx.x % LPG == LPG - 1;
    float w[R * 4];
#pragma unroll
    for (int k = 0; k < R * 4; ++k) {               // back by a slot, so that what is left is a turn forward
        const float before = __shfl_sync(0xffffffffu, last ? v[(k + 4 * R - 4) % (4 * R)] : v[k], neighbour<LPG>(LPG - 1));
        w[k] = from < to ? before : v[k];
    }
    const int by = from - to & 3;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float all[7], half[6];
#pragma unroll
        for (int i = 0; i < 4; ++i) all[i] = w[4 * r + i];
#pragma unroll
        for (int i = 0; i < 3; ++i) all[4 + i] = __shfl_sync(0xffffffffu, first ? w[(4 * r + 4) % (4 * R) + i] : w[4 * r + i], neighbour<LPG>(1));
#pragma unroll
        for (int i = 0; i < 6; ++i) half[i] = by & 1 ? all[i + 1 < 7 ? i + 1 : 6] : all[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * r + i] = by & 2 ? half[i + 2] : half[i];
    }
}

template <int ACCESS> constexpr bool kAhead = ACCESS != TURNED;
constexpr int kAheadBlocks = 16;        // blocks an SM of the kernels that take several tiles

// Five blocks an SM where registers hold that: 232965 x 602 fp32 162 -> 152 us, bf16 SiLU of 169343 x 601 177 -> 174 (six: 153, 219).
// In the other rows the compiler is asked for one block with an activation, for nothing (0) without: one block means 106 registers in
// place of 80.  Packing 100000 x 500 in groups of 100 61 us against 84, x 1024 in one 134 against 203; GELU of the second 250 against 226.
template <class T, int ACCESS, int LPG, int R, bool ACT>
__global__ void __launch_bounds__(kBlock, ACCESS == TURNED ? (R <= 4 ? 5 : 1) : ACT ? 1 : 0) rows8_pack_kernel(const __grid_constant__ Rows8Args a) {
    constexpr int U = Tile<LPG, R>::U, NG = Tile<LPG, R>::kGroups;
    const int job = blockIdx.x % a.jobs, lane = threadIdx.x % LPG;
    const T *x = static_cast<const T *>(a.x[job]);
    const int run = a.run[job];
    float ahead[U][R * 4];
    Where to_come[U];
    const auto fetch = [&](int64_t tile) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = tile * (NG * U) + threadIdx.x / LPG + u * NG;
            to_come[u] = {0, 0, 0, 0};
            if (i < a.items) to_come[u] = locate(a, i, a.ldx[job]);
            load_group<T, ACCESS, LPG, R>(x + to_come[u].x, to_come[u].n, x, x + (a.rows - 1) * a.ldx[job] + a.cols, ahead[u]);
        }
    };
    // Where registers allow, a block takes several tiles and has the next one's loads under way: 100000 x 500 in groups of 100
    // 78 -> 67 us (61 with the other blocks as they are now).  (In turned rows it lost: 232965 x 602 166 -> 203.)
    int64_t tile = blockIdx.x / a.jobs;
    const int64_t tiles = (a.items + NG * U - 1) / (NG * U), apart = gridDim.x / a.jobs;
    fetch(tile);
    do {
        const int64_t first = tile * (NG * U) + threadIdx.x / LPG;
        float v[U][R * 4];
        Where w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            w[u] = to_come[u];
#pragma unroll
            for (int k = 0; k < R * 4; ++k) v[u][k] = ahead[u][k];
        }
        tile += apart;
        if (kAhead<ACCESS> && tile < tiles) fetch(tile);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float top = 0.f;
#pragma unroll
            for (int k = 0; k < R * 4; k += 2) top = max_abs3(v[u][k], v[u][k + 1], top);
#pragma unroll
            for (int o = LPG / 2; o > 0; o >>= 1) top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
            const int64_t i = first + u * NG;
            const bool keep = !ACT || a.q[job];          // an activation without a backward pass keeps nothing
            const int skip = skip_of<T, ACCESS>(x + w[u].x);
            if (keep) {
                const float s = group_scale(top), inv = group_inverse(s);
                const int width = code_width(a, w[u]);
                int8_t *q = a.q[job] + (code_place(a, w[u]) << (run > 0));
                if (lane == 0 && i < a.items) a.scale[job][i * a.scale_stride[job]] = s;
                uint32_t word[R];
                if (a.mode == TANGO_ROUND_NEAREST) {
                    encode_nearest<R>(v[u], s, inv, word);
                } else {
#pragma unroll
                    for (int r = 0; r < R; ++r)
                        word[r] = encode4_mode(four(v[u] + 4 * r), s, a.mode, a.seed, effective_call(a.call + job, a.step),
                                               (uint64_t)w[u].row * a.cols + (int64_t)w[u].g * a.group + (lane + r * LPG) * 4 - skip,
                                               lane + r == 0 ? skip : 0, kSlots<LPG, R>);
                }
                if constexpr (ACCESS == TURNED) turn_back<LPG, R>(word, skip);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const int e = (lane + r * LPG) * 4;
                    if (e < width && i < a.items) *reinterpret_cast<uint32_t *>(q + (run ? ((e & -run) << 1 | (e & (run - 1))) : e)) = word[r];
                }
            }
            if constexpr (ACT) {
                with_act(a.act, [&](auto kind) {
#pragma unroll
                    for (int k = 0; k < R * 4; ++k) v[u][k] = activate<kind.value>(v[u][k]);
                });
                T *y = static_cast<T *>(a.y) + (w[u].x + w[u].row * (a.ldy - a.ldx[0]));
                if (ACCESS == TURNED && a.over) turn_over<LPG, R>(v[u], skip, skip_of<T, ACCESS>(y));
                store_group<T, ACCESS, LPG, R>(y, w[u].n, v[u]);
            }
        }
    } while (kAhead<ACCESS> && tile < tiles);
}

template <class T, int ACCESS, int LPG, int R, bool ACT>
__global__ void __launch_bounds__(kBlock) rows8_unpack_kernel(const __grid_constant__ Rows8Args a) {
    constexpr int U = Tile<LPG, R>::U, NG = Tile<LPG, R>::kGroups;
    const int lane = threadIdx.x % LPG;
    const int64_t first = (int64_t)blockIdx.x * (NG * U) + threadIdx.x / LPG;
    uint32_t word[U][R];
    float dy[ACT ? U : 1][R * 4], s[U];
    Where w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t i = first + u * NG;
        w[u] = {0, 0, 0, 0};
        if (i < a.items) w[u] = locate(a, i, a.ldy);
        s[u] = i < a.items ? __ldg(a.scale[0] + i) : 0.f;
        const int8_t *q = a.q[0] + code_place(a, w[u]) + lane * 4;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int e = (lane + r * LPG) * 4;
            word[u][r] = e < w[u].n ? __ldg(reinterpret_cast<const uint32_t *>(q + r * LPG * 4)) : 0u;
        }
        if constexpr (ACT) {
            const T *x = static_cast<const T *>(a.x[0]);
            load_group<T, ACCESS, LPG, R>(x + (w[u].x + w[u].row * (a.ldx[0] - a.ldy)), w[u].n, x, x + (a.rows - 1) * a.ldx[0] + a.cols, dy[u]);
        }
    }
    float o[U][R * 4];
    int skip[U], skip_out[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        skip[u] = skip_out[u] = skip_of<T, ACCESS>(static_cast<T *>(a.y) + w[u].x);
        if (ACT) skip[u] = skip_of<T, ACCESS>(static_cast<const T *>(a.x[0]) + (w[u].x + w[u].row * (a.ldx[0] - a.ldy)));
        if constexpr (ACCESS == TURNED) turn<LPG, R>(word[u], skip[u]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            Pair lo, hi;
            decode4(word[u][r], lo, hi);
            const float2 l = both(mul2(lo, pair(s[u], s[u]))), h = both(mul2(hi, pair(s[u], s[u])));
            o[u][4 * r] = l.x; o[u][4 * r + 1] = l.y; o[u][4 * r + 2] = h.x; o[u][4 * r + 3] = h.y;
        }
    }
    if constexpr (ACT) {
        with_act(a.act, [&](auto kind) {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int k = 0; k < R * 4; ++k) o[u][k] = __fmul_rn(dy[u][k], slope_of<kind.value>(o[u][k]));
        });
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (ACT && ACCESS == TURNED && a.over) turn_over<LPG, R>(o[u], skip[u], skip_out[u]);
        store_group<T, ACCESS, LPG, R>(static_cast<T *>(a.y) + w[u].x, w[u].n, o[u]);
    }
}

// ---- contiguous matrices whose groups have 4, 8, .. 128 columns and fill their rows: one run of memory in every respect (groups,
// scales and codes follow one another), four times four elements a lane, whole lines per access
template <class T, int GL, bool ACT, bool PACK>
__global__ void __launch_bounds__(kBlock) rows8_flat_kernel(const __grid_constant__ Rows8Args a) {
    constexpr int R = 4;                        // GL: lanes of a group
    const int job = blockIdx.x % a.jobs;
    const int64_t total = a.rows * a.cols, at = ((int64_t)(blockIdx.x / a.jobs) * kBlock * R + (threadIdx.x & ~31) * R + (threadIdx.x & 31)) * 4;
    float v[R * 4];
    uint32_t word[R];
    float s[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t e = at + r * 128;
        const bool there = e < total;
        if constexpr (PACK || ACT) load4<T, 4>(static_cast<const T *>(a.x[job]) + e, there ? 4 : 0, v + 4 * r);
        if constexpr (!PACK) {
            word[r] = there ? __ldg(reinterpret_cast<const uint32_t *>(a.q[0] + e)) : 0u;
            s[r] = there ? __ldg(a.scale[0] + e / (GL * 4)) : 0.f;
        }
    }
    if constexpr (PACK) {
        const bool keep = !ACT || a.q[job];
        if (keep) {
            float top[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                top[r] = max_abs3(max_abs3(v[4 * r], v[4 * r + 1], v[4 * r + 2]), v[4 * r + 3], 0.f);
#pragma unroll
                for (int o = GL / 2; o > 0; o >>= 1) top[r] = max_or_nan(top[r], __shfl_xor_sync(0xffffffffu, top[r], o));
            }
            if constexpr (GL >= 4) {        // four lanes of a group divide for one of its four pieces each
                const int k = threadIdx.x & 3;
                const float mine = group_scale(k < 2 ? (k == 0 ? top[0] : top[1]) : (k == 2 ? top[2] : top[3]));
#pragma unroll
                for (int r = 0; r < R; ++r) s[r] = __shfl_sync(0xffffffffu, mine, (threadIdx.x & 28) | r);
            } else {
#pragma unroll
                for (int r = 0; r < R; ++r) s[r] = group_scale(top[r]);
            }
            if (a.mode == TANGO_ROUND_NEAREST) {
#pragma unroll
                for (int r = 0; r < R; ++r) encode_nearest<1>(v + 4 * r, s[r], group_inverse(s[r]), word + r);
            } else {
#pragma unroll
                for (int r = 0; r < R; ++r)
                    word[r] = encode4_mode(four(v + 4 * r), s[r], a.mode, a.seed, effective_call(a.call + job, a.step), at + r * 128);
            }
            const int run = a.run[job];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int64_t e = at + r * 128;
                if (e >= total) continue;
                const int64_t q = run ? ((e & -(int64_t)run) << 1 | (e & (run - 1))) : e;
                *reinterpret_cast<uint32_t *>(a.q[job] + q) = word[r];
                if ((threadIdx.x & (GL - 1)) == 0) a.scale[job][e / (GL * 4) * a.scale_stride[job]] = s[r];
            }
        }
        if constexpr (ACT) {
            with_act(a.act, [&](auto kind) {
#pragma unroll
                for (int k = 0; k < R * 4; ++k) v[k] = activate<kind.value>(v[k]);
            });
#pragma unroll
            for (int r = 0; r < R; ++r)
                store4<T, 4>(static_cast<T *>(a.y) + at + r * 128, at + r * 128 < total ? 4 : 0, v + 4 * r);
        }
    } else {
        float o[R * 4];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            Pair lo, hi;
            decode4(word[r], lo, hi);
            const float2 l = both(mul2(lo, pair(s[r], s[r]))), h = both(mul2(hi, pair(s[r], s[r])));
            o[4 * r] = l.x; o[4 * r + 1] = l.y; o[4 * r + 2] = h.x; o[4 * r + 3] = h.y;
        }
        if constexpr (ACT) {
            with_act(a.act, [&](auto kind) {
#pragma unroll
                for (int k = 0; k < R * 4; ++k) o[k] = __fmul_rn(v[k], slope_of<kind.value>(o[k]));
            });
        }
#pragma unroll
        for (int r = 0; r < R; ++r) store4<T, 4>(static_cast<T *>(a.y) + at + r * 128, at + r * 128 < total ? 4 : 0, o + 4 * r);
    }
}

template <class T, int ACCESS, bool ACT, bool PACK, int LPG, int R>
static int launch_kernel(const Rows8Args &a, int jobs, cudaStream_t st) {
    int64_t blocks = ceil_div(a.items, Tile<LPG, R>::kItems);
    if (PACK && kAhead<ACCESS> && blocks > kNumSMs * kAheadBlocks) blocks = kNumSMs * kAheadBlocks;
    blocks *= jobs;
    if (blocks > 0x7fffffffLL) return TANGO_ESIZE;
    const unsigned grid = (unsigned)blocks;
    if constexpr (PACK) rows8_pack_kernel<T, ACCESS, LPG, R, ACT><<<grid, kBlock, 0, st>>>(a);
    else rows8_unpack_kernel<T, ACCESS, LPG, R, ACT><<<grid, kBlock, 0, st>>>(a);
    TANGO_LAUNCH_CHECK();
    return TANGO_OK;
}

template <class T, bool ACT, bool PACK, int GL>
static int launch_flat(const Rows8Args &a, int jobs, cudaStream_t st) {
    const int64_t blocks = ceil_div(a.rows * a.cols, kBlock * 16) * jobs;
    if (blocks > 0x7fffffffLL) return TANGO_ESIZE;
    rows8_flat_kernel<T, GL, ACT, PACK><<<(unsigned)blocks, kBlock, 0, st>>>(a);
    TANGO_LAUNCH_CHECK();
    return TANGO_OK;
}
template <class T, bool ACT, bool PACK>
static int launch_flat(const Rows8Args &a, int jobs, cudaStream_t st) {
    switch (a.group) {
        case 4: return launch_flat<T, ACT, PACK, 1>(a, jobs, st);
        case 8: return launch_flat<T, ACT, PACK, 2>(a, jobs, st);
        case 16: return launch_flat<T, ACT, PACK, 4>(a, jobs, st);
        case 32: return launch_flat<T, ACT, PACK, 8>(a, jobs, st);
        case 64: return launch_flat<T, ACT, PACK, 16>(a, jobs, st);
        default: return launch_flat<T, ACT, PACK, 32>(a, jobs, st);
    }
}

template <class T, int ACCESS, bool ACT, bool PACK>
static int launch_tile(const Rows8Args &a, int jobs, cudaStream_t st) {
    if (a.tile <= 4) return launch_kernel<T, ACCESS, ACT, PACK, 1, 1>(a, jobs, st);
    if (a.tile <= 8) return launch_kernel<T, ACCESS, ACT, PACK, 1, 2>(a, jobs, st);
    if (a.tile <= 16) return launch_kernel<T, ACCESS, ACT, PACK, 1, 4>(a, jobs, st);
    if (a.tile <= 32) return launch_kernel<T, ACCESS, ACT, PACK, 2, 4>(a, jobs, st);
    if (a.tile <= 64) return launch_kernel<T, ACCESS, ACT, PACK, 4, 4>(a, jobs, st);
    if (a.tile <= 128) return launch_kernel<T, ACCESS, ACT, PACK, 8, 4>(a, jobs, st);
    if (a.tile <= 256) return launch_kernel<T, ACCESS, ACT, PACK, 16, 4>(a, jobs, st);
    if (a.tile <= 512) return launch_kernel<T, ACCESS, ACT, PACK, 32, 4>(a, jobs, st);
    return launch_kernel<T, ACCESS, ACT, PACK, 32, 8>(a, jobs, st);
}

template <bool ACT, bool PACK>
static int launch(Rows8Args a, int jobs, int type, int access, cudaStream_t st) {
    a.jobs = jobs;
    const auto go = [&](auto t) {
        typedef decltype(t) T;
        if (access == FLAT) return launch_flat<T, ACT, PACK>(a, jobs, st);
        if (access == WIDE) return launch_tile<T, WIDE, ACT, PACK>(a, jobs, st);
        return launch_tile<T, TURNED, ACT, PACK>(a, jobs, st);
    };
    if (type == TANGO_FP32) return go(float{});
    if (type == TANGO_BF16) return go(Bf16{});
    return go(Fp16{});
}

static int64_t element_bytes(int type) { return type == TANGO_FP32 ? 4 : 2; }

static bool fits_32(int64_t v);
static int fill(Rows8Args &a, int64_t rows, int64_t cols, int64_t group, int type) {
    if (rows < 0 || cols < 0 || group < 1 || type < TANGO_FP32 || type > TANGO_FP16) return TANGO_EINVAL;
    if (group > kMaxGroup) return TANGO_ESIZE;
    if (rows == 0 || cols == 0) return TANGO_OK;
    const int64_t groups = ceil_div(cols, group);
    if (groups > 0x7fffffffLL || rows > INT64_MAX / groups) return TANGO_ESIZE;
    a.rows = rows; a.cols = cols; a.group = (int32_t)group; a.groups = (int32_t)groups;
    a.items = rows * groups;
    a.pitch = (int32_t)tango_rows8_pitch(group);
    a.ldq = tango_rows8_ld(cols, group);
    // a row of one group is shared out by its own length: 19717 x 64 in groups of up to 128, packed with
    // ELU, 9.5 -> 7.0 us
    a.tile = (int32_t)(groups == 1 && a.ldq < group ? a.ldq : group);
    if (groups == 1 && a.ldq == cols) a.group = (int32_t)cols;
    a.wide = !fits_32(a.items) || !fits_32(cols);
    a.by_groups = fast_div(groups);
    return TANGO_OK;
}

// What the matrices of a launch, with their leading dimensions, allow.
static int access_of(const Rows8Args &a, int type, std::initializer_list<const void *> matrices, std::initializer_list<int64_t> lds) {
    bool wide = a.groups == 1 || a.group % 4 == 0, run = a.ldq == a.cols;
    for (const void *p : matrices) wide &= aligned(p, 4 * element_bytes(type));
    for (int64_t ld : lds) { wide &= a.rows == 1 || ld % 4 == 0; run &= a.rows == 1 || ld == a.cols; }
    if (wide && run && a.cols % a.group == 0 && a.group <= 128 && a.group >= 4 && (a.group & (a.group - 1)) == 0) return FLAT;
    return wide ? WIDE : TURNED;
}
static int lie_apart(const Rows8Args &a, int type) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.x[0]), y = reinterpret_cast<uintptr_t>(a.y), e = (uintptr_t)element_bytes(type);
    return (x / e & 3) != (y / e & 3) || (a.rows > 1 && (a.ldx[0] - a.ldy) % 4 != 0);
}
static bool fits_32(int64_t v) { return v < 0x7fffffffLL; }

}  // namespace tango

using namespace tango;

extern "C" int64_t tango_rows8_run(int64_t group) { return group < 1 ? TANGO_EINVAL : group > 8 ? 16 : group > 4 ? 8 : 4; }

extern "C" int64_t tango_rows8_pitch(int64_t group) { return group < 1 ? TANGO_EINVAL : round_up(group, tango_rows8_run(group)); }

extern "C" int64_t tango_rows8_ld(int64_t cols, int64_t group) {
    if (cols < 0 || group < 1) return TANGO_EINVAL;
    if (cols == 0) return 0;
    const int64_t before = (cols - 1) / group;
    return before * tango_rows8_pitch(group) + round_up(cols - before * group, tango_rows8_run(group));
}

extern "C" int tango_rows8_pack(const tango_rows8_job *jobs, int n_jobs, int64_t rows, int64_t cols, int64_t group, int type,
                                int mode, uint64_t seed, uint64_t call, const uint64_t *step, tango_stream_t stream) {
    if (!jobs || n_jobs < 1 || n_jobs > kMaxJobs || mode < TANGO_ROUND_TRUNC || mode > TANGO_ROUND_STOCHASTIC) return TANGO_EINVAL;
    Rows8Args a{};
    const int rc = fill(a, rows, cols, group, type);
    if (rc != TANGO_OK || rows == 0 || cols == 0) return rc;
    int access = FLAT;
    for (int k = 0; k < n_jobs; ++k) {
        const tango_rows8_job &j = jobs[k];
        if (!j.x || !j.q || !j.scales || j.scale_stride < 1 || (rows > 1 && j.ldx < cols)) return TANGO_EINVAL;
        if (!aligned(j.x, element_bytes(type)) || !aligned(j.q, 4)) return TANGO_EALIGN;
        a.x[k] = j.x; a.ldx[k] = j.ldx; a.q[k] = j.q; a.scale[k] = j.scales;
        a.scale_stride[k] = j.scale_stride;
        a.run[k] = j.interleaved ? (int)tango_rows8_run(group) : 0;
        a.wide |= !fits_32(j.ldx);
        const int way = access_of(a, type, {j.x}, {j.ldx});
        if (way < access) access = way;
    }
    a.mode = mode; a.act = ACT_NONE; a.seed = seed; a.call = call;
    a.step = reinterpret_cast<const unsigned long long *>(step);
    return launch<false, true>(a, n_jobs, type, access, static_cast<cudaStream_t>(stream));
}

extern "C" int tango_rows8_unpack(const int8_t *q, const float *scales, int64_t rows, int64_t cols, int64_t group, int type,
                                  void *out, int64_t ldo, tango_stream_t stream) {
    Rows8Args a{};
    const int rc = fill(a, rows, cols, group, type);
    if (rc != TANGO_OK || rows == 0 || cols == 0) return rc;
    if (!q || !scales || !out || (rows > 1 && ldo < cols)) return TANGO_EINVAL;
    if (!aligned(out, element_bytes(type)) || !aligned(q, 4)) return TANGO_EALIGN;
    a.q[0] = const_cast<int8_t *>(q); a.scale[0] = const_cast<float *>(scales); a.y = out; a.ldy = ldo; a.act = ACT_NONE;
    a.wide |= !fits_32(ldo);
    return launch<false, false>(a, 1, type, access_of(a, type, {out}, {ldo}), static_cast<cudaStream_t>(stream));
}

extern "C" int tango_act8_forward(int act, const tango_rows8_job *job, int64_t rows, int64_t cols, int64_t group, int type, void *y,
                                  int64_t ldy, int mode, uint64_t seed, uint64_t call, const uint64_t *step, tango_stream_t stream) {
    if (!job || act < ACT_ELU || act > ACT_SILU || mode < TANGO_ROUND_TRUNC || mode > TANGO_ROUND_STOCHASTIC) return TANGO_EINVAL;
    Rows8Args a{};
    const int rc = fill(a, rows, cols, group, type);
    if (rc != TANGO_OK || rows == 0 || cols == 0) return rc;
    if (!job->x || !job->q != !job->scales || (job->q && job->scale_stride < 1) || !y || (rows > 1 && (job->ldx < cols || ldy < cols))) return TANGO_EINVAL;
    if (!aligned(job->x, element_bytes(type)) || !aligned(y, element_bytes(type)) || !aligned(job->q, 4)) return TANGO_EALIGN;
    a.x[0] = job->x; a.ldx[0] = job->ldx; a.q[0] = job->q; a.scale[0] = job->scales; a.scale_stride[0] = job->scale_stride; a.y = y; a.ldy = ldy;
    a.wide |= !fits_32(job->ldx) || !fits_32(ldy);
    a.over = lie_apart(a, type);
    a.mode = mode; a.act = act; a.seed = seed; a.call = call;
    a.step = reinterpret_cast<const unsigned long long *>(step);
    return launch<true, true>(a, 1, type, access_of(a, type, {job->x, y}, {job->ldx, ldy}), static_cast<cudaStream_t>(stream));
}

extern "C" int tango_act8_backward(int act, const int8_t *q, const float *scales, int64_t rows, int64_t cols, int64_t group, int type,
                                   const void *dy, int64_t lddy, void *dx, int64_t lddx, tango_stream_t stream) {
    if (act < ACT_ELU || act > ACT_SILU) return TANGO_EINVAL;
    Rows8Args a{};
    const int rc = fill(a, rows, cols, group, type);
    if (rc != TANGO_OK || rows == 0 || cols == 0) return rc;
    if (!q || !scales || !dy || !dx || (rows > 1 && (lddy < cols || lddx < cols))) return TANGO_EINVAL;
    if (!aligned(dy, element_bytes(type)) || !aligned(dx, element_bytes(type)) || !aligned(q, 4)) return TANGO_EALIGN;
    a.q[0] = const_cast<int8_t *>(q); a.scale[0] = const_cast<float *>(scales);
    a.x[0] = dy; a.ldx[0] = lddy; a.y = dx; a.ldy = lddx; a.act = act;
    a.wide |= !fits_32(lddy) || !fits_32(lddx);
    a.over = lie_apart(a, type);
    return launch<true, false>(a, 1, type, access_of(a, type, {dy, dx}, {lddy, lddx}), static_cast<cudaStream_t>(stream));
}
