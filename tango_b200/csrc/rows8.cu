// 8-bit rows: packing, unpacking, and activations whose saved input is held in them.
//
//   pack     : s = max|x| / 127 over a group, codes x / s exactly rounded; with an activation also y = f(x) in the same pass
//   unpack   : code * s
//   backward : dx = dy * f'(code * s), from the 8-bit copy alone
//
// Bound by HBM: pack 5 bytes an fp32 element (4 read, 1 written), unpack 5, activation forward 9, backward 9.  A group is
// owned by a few lanes, each with R times four neighbouring elements LPG * 4 apart (a load and the store of four codes are
// contiguous over the lanes), so that x is read once and stays in registers.
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
    int64_t ldq;
    FastDiv by_groups;
    int wide;                     // 2^31 groups or more
    int mode, act;
    uint64_t seed, call;
    const unsigned long long *step;
};

template <int K> struct Kind { static constexpr int value = K; };

__device__ __forceinline__ float exp_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
    return y;
}
// Upper tail of the normal distribution at |x| times two, erfc(|x| / sqrt(2)), with e = exp(-x^2 / 2): the rational formula 7.1.26
// of Abramowitz and Stegun's handbook (|error| < 1.5e-7), which shares the exponential with the density.
__device__ __forceinline__ float normal_tails(float x, float e) {
    const float t = __fdividef(1.f, fmaf(0.3275911f * 0.70710678118654752f, fabsf(x), 1.f));
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
    return __fdividef(x, 1.f + exp_fast(-x));
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
    const float s = __fdividef(1.f, 1.f + exp_fast(-t));
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

template <class T, int VL, int LPG, int R, bool ACT>
__global__ void __launch_bounds__(kBlock) rows8_pack_kernel(const __grid_constant__ Rows8Args a) {
    constexpr int U = Tile<LPG, R>::U, NG = Tile<LPG, R>::kGroups;
    const int job = blockIdx.y, lane = threadIdx.x % LPG;
    const T *x = static_cast<const T *>(a.x[job]);
    const int64_t first = (int64_t)blockIdx.x * (NG * U) + threadIdx.x / LPG;
    float v[U][R * 4];
    Where w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t i = first + u * NG;
        w[u] = {0, 0, 0, 0};
        if (i < a.items) w[u] = locate(a, i, a.ldx[job]);
        const T *p = x + w[u].x + lane * 4;
#pragma unroll
        for (int r = 0; r < R; ++r) load4<T, VL>(p + r * LPG * 4, w[u].n - (lane + r * LPG) * 4, v[u] + 4 * r);
    }
    const int run = a.run[job];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < R * 4; k += 2) top = max_abs3(v[u][k], v[u][k + 1], top);
#pragma unroll
        for (int o = LPG / 2; o > 0; o >>= 1) top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
        const int64_t i = first + u * NG;
        if (i >= a.items) continue;
        const bool keep = !ACT || a.q[job];          // an activation without a backward pass keeps nothing
        if (keep) {
            const float s = group_scale(top), inv = group_inverse(s);
            const int width = code_width(a, w[u]);
            int8_t *q = a.q[job] + (code_place(a, w[u]) << (run > 0));
            if (lane == 0) a.scale[job][i * a.scale_stride[job]] = s;
            uint32_t word[R];
            if (a.mode == TANGO_ROUND_NEAREST) {
                encode_nearest<R>(v[u], s, inv, word);
            } else {
#pragma unroll
                for (int r = 0; r < R; ++r)
                    word[r] = encode4_mode(v[u] + 4 * r, s, a.mode, a.seed, effective_call(a.call + job, a.step),
                                           (uint64_t)w[u].row * a.cols + (int64_t)w[u].g * a.group + (lane + r * LPG) * 4);
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int e = (lane + r * LPG) * 4;
                if (e < width) *reinterpret_cast<uint32_t *>(q + (run ? ((e & -run) << 1 | (e & (run - 1))) : e)) = word[r];
            }
        }
        if constexpr (ACT) {
            T *y = static_cast<T *>(a.y) + (w[u].x + w[u].row * (a.ldy - a.ldx[0])) + lane * 4;
            with_act(a.act, [&](auto kind) {
#pragma unroll
                for (int k = 0; k < R * 4; ++k) v[u][k] = activate<kind.value>(v[u][k]);
            });
#pragma unroll
            for (int r = 0; r < R; ++r) store4<T, VL>(y + r * LPG * 4, w[u].n - (lane + r * LPG) * 4, v[u] + 4 * r);
        }
    }
}

template <class T, int VL, int LPG, int R, bool ACT>
__global__ void __launch_bounds__(kBlock) rows8_unpack_kernel(const __grid_constant__ Rows8Args a) {
    constexpr int U = Tile<LPG, R>::U, NG = Tile<LPG, R>::kGroups;
    const int lane = threadIdx.x % LPG;
    const int64_t first = (int64_t)blockIdx.x * (NG * U) + threadIdx.x / LPG;
    uint32_t word[U][R];
    float dy[ACT ? U : 1][R][4], s[U];
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
            if constexpr (ACT)
                load4<T, VL>(static_cast<const T *>(a.x[0]) + (w[u].x + w[u].row * (a.ldx[0] - a.ldy)) + e, w[u].n - e, dy[u][r]);
        }
    }
    float o[U][R][4];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            Pair lo, hi;
            decode4(word[u][r], lo, hi);
            const float2 l = both(mul2(lo, pair(s[u], s[u]))), h = both(mul2(hi, pair(s[u], s[u])));
            o[u][r][0] = l.x; o[u][r][1] = l.y; o[u][r][2] = h.x; o[u][r][3] = h.y;
        }
    if constexpr (ACT) {
        with_act(a.act, [&](auto kind) {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int k = 0; k < 4; ++k) o[u][r][k] = __fmul_rn(dy[u][r][k], slope_of<kind.value>(o[u][r][k]));
        });
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int e = (lane + r * LPG) * 4;
            store4<T, VL>(static_cast<T *>(a.y) + w[u].x + e, w[u].n - e, o[u][r]);
        }
}

// ---- contiguous matrices whose groups have 4, 8, .. 128 columns and fill their rows: one run of memory in every respect (groups,
// scales and codes follow one another), four times four elements a lane, whole lines per access
template <class T, int GL, bool ACT, bool PACK>
__global__ void __launch_bounds__(kBlock) rows8_flat_kernel(const __grid_constant__ Rows8Args a) {
    constexpr int R = 4;                        // GL: lanes of a group
    const int job = blockIdx.y;
    const int64_t total = a.rows * a.cols, at = ((int64_t)blockIdx.x * kBlock * R + (threadIdx.x & ~31) * R + (threadIdx.x & 31)) * 4;
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
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float top = max_abs3(v[4 * r], v[4 * r + 1], 0.f);
                top = max_abs3(v[4 * r + 2], v[4 * r + 3], top);
#pragma unroll
                for (int o = GL / 2; o > 0; o >>= 1) top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
                s[r] = group_scale(top);
            }
            if (a.mode == TANGO_ROUND_NEAREST) {
#pragma unroll
                for (int r = 0; r < R; ++r) encode_nearest<1>(v + 4 * r, s[r], group_inverse(s[r]), word + r);
            } else {
#pragma unroll
                for (int r = 0; r < R; ++r)
                    word[r] = encode4_mode(v + 4 * r, s[r], a.mode, a.seed, effective_call(a.call + job, a.step), at + r * 128);
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

// ---- contiguous matrices whose row pitch allows no wide access (601 columns): the items of a block are one run of memory all the
// same, in the matrix as in the codes, and pass through shared memory in 16-byte pieces, the next ones while a block works on
// one.  Lanes take single neighbouring elements there.
__device__ __forceinline__ void copy_async(void *shared, const void *global) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(shared)), "l"(global) : "memory");
}
// from[begin .. begin + n) of an array of `total` elements to to[begin % per ..], by whole 16-byte pieces of the array (which its
// last elements may not fill).
template <class T>
__device__ __forceinline__ void copy_in(T *to, const T *from, int64_t begin, int n, int64_t total) {
    constexpr int per = 16 / sizeof(T);
    const int lead = (int)(begin & (per - 1));
    const T *p = from + (begin - lead);
    const int64_t left = total - (begin - lead);
    for (int at = threadIdx.x * per; at < lead + n; at += kBlock * per) {
        if (at + per <= left) {
            copy_async(to + at, p + at);
        } else {
            for (int k = at; k < left; ++k) to[k] = p[k];
        }
    }
}
template <class T>
__device__ __forceinline__ void copy_out(T *to, int64_t begin, int n, const T *from) {
    constexpr int per = 16 / sizeof(T);
    const int lead = (int)(begin & (per - 1));
    T *p = to + (begin - lead);
    const int end = lead + n;
    for (int at = threadIdx.x * per; at < end; at += kBlock * per) {
        if (at >= lead && at + per <= end) {
            *reinterpret_cast<uint4 *>(p + at) = *reinterpret_cast<const uint4 *>(from + at);
        } else {
            for (int k = at < lead ? lead : at; k < at + per && k < end; ++k) p[k] = from[k];
        }
    }
}

// The run of a block's items: first element and byte of codes, and how many of each.
struct Run {
    int64_t x, q;
    int n, nq, items;
};
__device__ __forceinline__ Run run_of(const Rows8Args &a, int items, int64_t first) {
    Run r;
    r.items = a.items - first < items ? (int)(a.items - first) : items;
    const Where b = locate(a, first, a.cols), e = locate(a, first + r.items - 1, a.cols);
    r.x = b.x; r.n = (int)(e.x + e.n - b.x);
    r.q = code_place(a, b); r.nq = (int)(code_place(a, e) + code_width(a, e) - r.q);
    return r;
}

// The r-th element of this lane's group: neighbouring lanes, neighbouring elements, and every group of a warp begins at another
// place (32 elements are one turn of all banks), for groups that start in one bank of shared memory.
template <int LPG, int R>
__device__ __forceinline__ int turned(int r) { return ((int)(threadIdx.x % 32) + r * LPG) & (LPG * R * 4 - 1); }

// Shared memory: buffers of elements and of codes, each with room for the pieces that stick out at both ends.
template <class T, int LPG, int R, bool ACT, bool PACK> struct Staging {
    static constexpr int kX = (Tile<LPG, R>::kElements + 32 / (int)sizeof(T)) * (int)sizeof(T), kQ = Tile<LPG, R>::kElements + 32;
    static constexpr int kXs = PACK || ACT ? 2 : 1, kQs = PACK ? 1 : 2;
    static constexpr int kBytes = kXs * kX + kQs * kQ;
};

template <class T, int LPG, int R, bool ACT, bool PACK>
__global__ void __launch_bounds__(kBlock, 4) rows8_staged_kernel(const __grid_constant__ Rows8Args a) {
    typedef Tile<LPG, R> Shape;
    typedef Staging<T, LPG, R, ACT, PACK> Room;
    extern __shared__ __align__(16) char room[];
    const int job = blockIdx.y, lane = threadIdx.x % LPG;
    const int64_t tiles = (a.items + Shape::kItems - 1) / Shape::kItems, total = a.rows * a.cols, total_q = a.rows * a.ldq;
    const auto buffer_x = [&](int64_t t) { return reinterpret_cast<T *>(room + (Room::kXs > 1 ? (t & 1) * Room::kX : 0)); };
    const auto buffer_q = [&](int64_t t) {
        return reinterpret_cast<int8_t *>(room + Room::kXs * Room::kX + (Room::kQs > 1 ? (t & 1) * Room::kQ : 0));
    };
    const auto fetch = [&](int64_t tile, int64_t t) {
        Run run{};
        if (tile < tiles) {
            run = run_of(a, Shape::kItems, tile * Shape::kItems);
            if constexpr (PACK || ACT) copy_in(buffer_x(t), static_cast<const T *>(a.x[job]), run.x, run.n, total);
            if constexpr (!PACK) copy_in(buffer_q(t), a.q[0], run.q, run.nq, total_q);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        return run;
    };
    const bool keep = !PACK || !ACT || a.q[job];
    Run next = fetch(blockIdx.x, 0);
    for (int64_t t = 0, tile = blockIdx.x; tile < tiles; ++t, tile += gridDim.x) {
        const Run run = next;
        next = fetch(tile + gridDim.x, t + 1);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncthreads();
        const int64_t first = tile * Shape::kItems;
        T *s_x = buffer_x(t);
        int8_t *s_q = buffer_q(t);
        const int lead = (int)(run.x & (16 / sizeof(T) - 1)), lead_q = (int)(run.q & 15);
#pragma unroll
        for (int u = 0; u < Shape::U; ++u) {
            const int k = threadIdx.x / LPG + u * Shape::kGroups;
            const bool there = k < run.items;
            Where w = {0, 0, 0, 0};
            if (there) w = locate(a, first + k, a.cols);
            // threads without an item read along with the first one
            T *x = s_x + lead + (there ? (int)(w.x - run.x) : 0);
            int8_t *q = s_q + lead_q + (there ? (int)(code_place(a, w) - run.q) : 0);
            if constexpr (PACK) {
                // elements behind the item's end are read too (they are in the buffer) and taken for 0
                float v[R * 4], top = 0.f;
#pragma unroll
                for (int r = 0; r < R * 4; ++r) v[r] = to_float(x[turned<LPG, R>(r)]);
#pragma unroll
                for (int r = 0; r < R * 4; ++r) v[r] = turned<LPG, R>(r) < w.n ? v[r] : 0.f;
#pragma unroll
                for (int r = 0; r < R * 4; r += 2) top = max_abs3(v[r], v[r + 1], top);
#pragma unroll
                for (int o = LPG / 2; o > 0; o >>= 1) top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
                if (there && keep) {
                    const float s = group_scale(top), inv = group_inverse(s);
                    if (lane == 0) a.scale[job][(first + k) * a.scale_stride[job]] = s;
                    const int width = code_width(a, w);
                    if (a.mode == TANGO_ROUND_NEAREST) {
                        float b[R * 4];
                        round_nearest<R * 4>(v, s, inv, b);
#pragma unroll
                        for (int r = 0; r < R * 4; ++r) {
                            const int e = turned<LPG, R>(r);
                            if (e < width) q[e] = inv == 0.f ? (int8_t)0 : (int8_t)__float_as_uint(b[r]);
                        }
                    } else {
#pragma unroll 1
                        for (int r = 0; r < R * 4; ++r) {
                            const int e = turned<LPG, R>(r);
                            if (e < width)
                                q[e] = e < w.n ? (int8_t)encode_mode(to_float(x[e]), s, a.mode, a.seed, effective_call(a.call + job, a.step),
                                                                     (uint64_t)w.row * a.cols + (int64_t)w.g * a.group + e)
                                               : (int8_t)0;
                        }
                    }
                }
                if constexpr (ACT) {
                    with_act(a.act, [&](auto kind) {
#pragma unroll
                        for (int r = 0; r < R * 4; ++r) v[r] = activate<kind.value>(v[r]);
                    });
#pragma unroll
                    for (int r = 0; r < R * 4; ++r)
                        if (turned<LPG, R>(r) < w.n) from_float(v[r], x[turned<LPG, R>(r)]);
                }
            } else if (there) {
                const float s = __ldg(a.scale[0] + first + k);
                float o[R * 4];
#pragma unroll
                for (int r = 0; r < R * 4; ++r) o[r] = __fmul_rn((float)q[turned<LPG, R>(r)], s);
                if constexpr (ACT) {
                    float dy[R * 4];
#pragma unroll
                    for (int r = 0; r < R * 4; ++r) dy[r] = to_float(x[turned<LPG, R>(r)]);
                    with_act(a.act, [&](auto kind) {
#pragma unroll
                        for (int r = 0; r < R * 4; ++r) o[r] = __fmul_rn(dy[r], slope_of<kind.value>(o[r]));
                    });
                }
#pragma unroll
                for (int r = 0; r < R * 4; ++r)
                    if (turned<LPG, R>(r) < w.n) from_float(o[r], x[turned<LPG, R>(r)]);
            }
        }
        __syncthreads();
        if constexpr (PACK) {
            if (keep) copy_out(a.q[job], run.q, run.nq, s_q);
        }
        if constexpr (!PACK || ACT) copy_out(static_cast<T *>(a.y), run.x, run.n, s_x);
        __syncthreads();          // before the buffers are filled again
    }
}

// How the elements are reached: four at a time, the same in one run, one at a time (rows of any pitch), or through shared memory.
enum { SINGLE = 0, STAGED = 1, WIDE = 2, FLAT = 3 };

static int sm_count() {
    int device = 0, n = kNumSMs;
    if (cudaGetDevice(&device) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device);
    return n;
}

template <class T, int ACCESS, bool ACT, bool PACK, int LPG, int R>
static int launch_kernel(const Rows8Args &a, int jobs, cudaStream_t st) {
    const int64_t blocks = ceil_div(a.items, Tile<LPG, R>::kItems);
    if (blocks > 0x7fffffffLL) return TANGO_ESIZE;
    const dim3 grid((unsigned)blocks, (unsigned)jobs);
    if constexpr (ACCESS == STAGED) {
        constexpr int bytes = Staging<T, LPG, R, ACT, PACK>::kBytes, resident = 220 * 1024 / bytes < 4 ? 220 * 1024 / bytes : 4;
        const auto kernel = rows8_staged_kernel<T, LPG, R, ACT, PACK>;
        if (bytes > 48 * 1024) TANGO_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        const int64_t most = (int64_t)sm_count() * resident;
        kernel<<<dim3((unsigned)(blocks < most ? blocks : most), (unsigned)jobs), kBlock, bytes, st>>>(a);
    } else if constexpr (PACK) {
        rows8_pack_kernel<T, ACCESS == WIDE ? 4 : 1, LPG, R, ACT><<<grid, kBlock, 0, st>>>(a);
    } else {
        rows8_unpack_kernel<T, ACCESS == WIDE ? 4 : 1, LPG, R, ACT><<<grid, kBlock, 0, st>>>(a);
    }
    TANGO_LAUNCH_CHECK();
    return TANGO_OK;
}

template <class T, bool ACT, bool PACK, int GL>
static int launch_flat(const Rows8Args &a, int jobs, cudaStream_t st) {
    const int64_t blocks = ceil_div(a.rows * a.cols, kBlock * 16);
    if (blocks > 0x7fffffffLL) return TANGO_ESIZE;
    rows8_flat_kernel<T, GL, ACT, PACK><<<dim3((unsigned)blocks, (unsigned)jobs), kBlock, 0, st>>>(a);
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
    if (a.group <= 4) return launch_kernel<T, ACCESS, ACT, PACK, 1, 1>(a, jobs, st);
    if (a.group <= 8) return launch_kernel<T, ACCESS, ACT, PACK, 1, 2>(a, jobs, st);
    if (a.group <= 16) return launch_kernel<T, ACCESS, ACT, PACK, 1, 4>(a, jobs, st);
    if (a.group <= 32) return launch_kernel<T, ACCESS, ACT, PACK, 2, 4>(a, jobs, st);
    if (a.group <= 64) return launch_kernel<T, ACCESS, ACT, PACK, 4, 4>(a, jobs, st);
    if (a.group <= 128) return launch_kernel<T, ACCESS, ACT, PACK, 8, 4>(a, jobs, st);
    if (a.group <= 256) return launch_kernel<T, ACCESS, ACT, PACK, 16, 4>(a, jobs, st);
    if (a.group <= 512) return launch_kernel<T, ACCESS, ACT, PACK, 32, 4>(a, jobs, st);
    return launch_kernel<T, ACCESS, ACT, PACK, 32, 8>(a, jobs, st);
}

template <bool ACT, bool PACK>
static int launch(const Rows8Args &a, int jobs, int type, int access, cudaStream_t st) {
    const auto go = [&](auto t) {
        typedef decltype(t) T;
        return access == FLAT     ? launch_flat<T, ACT, PACK>(a, jobs, st)
               : access == WIDE   ? launch_tile<T, WIDE, ACT, PACK>(a, jobs, st)
               : access == STAGED ? launch_tile<T, STAGED, ACT, PACK>(a, jobs, st)
                                  : launch_tile<T, SINGLE, ACT, PACK>(a, jobs, st);
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
    a.wide = !fits_32(a.items) || !fits_32(cols);
    a.by_groups = fast_div(groups);
    return TANGO_OK;
}

// What the matrices (with their leading dimensions) and the codes of a launch allow.
static int access_of(const Rows8Args &a, int type, std::initializer_list<const void *> matrices, std::initializer_list<int64_t> lds,
                     std::initializer_list<const void *> codes, bool interleaved) {
    bool wide = a.groups == 1 || a.group % 4 == 0, run = true, pieces = true;
    for (const void *p : matrices) { wide &= aligned(p, 4 * element_bytes(type)); pieces &= aligned(p, 16); }
    for (int64_t ld : lds) { wide &= a.rows == 1 || ld % 4 == 0; run &= a.rows == 1 || ld == a.cols; }
    for (const void *p : codes) pieces &= aligned(p, 16);
    if (wide && run && a.cols % a.group == 0 && a.group <= 128 && a.group >= 4 && (a.group & (a.group - 1)) == 0) return FLAT;
    if (wide) return WIDE;
    return run && pieces && !interleaved ? STAGED : SINGLE;
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
        const int way = access_of(a, type, {j.x}, {j.ldx}, {j.q}, j.interleaved);
        if (way < access) access = way;
    }
    // what one of them cannot do is done by none; the staged form asks for more than the wide one
    for (int k = 0; k < n_jobs && access == STAGED; ++k)
        if (!aligned(jobs[k].x, 16) || (rows > 1 && jobs[k].ldx != cols) || !aligned(jobs[k].q, 16) || jobs[k].interleaved) access = SINGLE;
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
    return launch<false, false>(a, 1, type, access_of(a, type, {out}, {ldo}, {q}, false), static_cast<cudaStream_t>(stream));
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
    a.mode = mode; a.act = act; a.seed = seed; a.call = call;
    a.step = reinterpret_cast<const unsigned long long *>(step);
    return launch<true, true>(a, 1, type, access_of(a, type, {job->x, y}, {job->ldx, ldy}, {job->q}, false), static_cast<cudaStream_t>(stream));
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
    return launch<true, false>(a, 1, type, access_of(a, type, {dy, dx}, {lddy, lddx}, {q}, false), static_cast<cudaStream_t>(stream));
}
