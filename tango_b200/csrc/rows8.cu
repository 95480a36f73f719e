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

__device__ __forceinline__ float activate(float x, int act) {
    if (act == ACT_ELU) return x > 0.f ? x : expm1f(x);
    if (act == ACT_GELU) return 0.5f * x * (1.f + erff(0.70710678118654752f * x));
    return __fdividef(x, 1.f + expf(-x));
}
// The slope is taken at the 8-bit copy, off by at most half a step; each f is smooth enough (|f''| <= 1, one-sided at ELU's 0,
// where the slope is continuous) that the slope moves by no more than that.
__device__ __forceinline__ float slope_of(float t, int act) {
    if (act == ACT_ELU) return t > 0.f ? 1.f : expf(t);
    if (act == ACT_GELU) return fmaf(t * 0.39894228040143268f, expf(-0.5f * t * t), 0.5f * (1.f + erff(0.70710678118654752f * t)));
    const float s = __fdividef(1.f, 1.f + expf(-t));
    return s == 0.f ? 0.f : s * fmaf(t, 1.f - s, 1.f);
}

// Where item `i` (a group of a row) lies.
struct Where {
    int64_t row;
    int32_t g, n;      // group, its elements
};
__device__ __forceinline__ Where locate(const Rows8Args &a, int64_t i) {
    Where w;
    if (a.wide) {
        w.row = i / a.groups;
        w.g = (int32_t)(i - w.row * a.groups);
    } else {
        const uint32_t r = quotient((uint32_t)i, a.by_groups);
        w.row = r;
        w.g = (int32_t)((uint32_t)i - r * (uint32_t)a.groups);
    }
    const int64_t left = a.cols - (int64_t)w.g * a.group;
    w.n = left < a.group ? (int32_t)left : a.group;
    return w;
}

// LPG lanes a group, R times four elements a lane, U groups in flight.
template <int LPG, int R> struct Tile {
    static constexpr int U = R == 1 ? 4 : R == 2 ? 2 : 1;
    static constexpr int kGroups = kBlock / LPG;        // groups a block works on at a time
};

template <class T, int VL, int LPG, int R, bool ACT>
__global__ void __launch_bounds__(kBlock) rows8_pack_kernel(const __grid_constant__ Rows8Args a) {
    constexpr int U = Tile<LPG, R>::U, NG = Tile<LPG, R>::kGroups;
    const int job = blockIdx.y, lane = threadIdx.x % LPG;
    const T *x = static_cast<const T *>(a.x[job]);
    const int64_t first = (int64_t)blockIdx.x * (NG * U) + threadIdx.x / LPG;
    float v[U][R][4];
    Where w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t i = first + u * NG;
        w[u] = {0, 0, 0};
        if (i < a.items) w[u] = locate(a, i);
        const T *p = x + w[u].row * a.ldx[job] + (int64_t)w[u].g * a.group;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int e = (lane + r * LPG) * 4;
            load4<T, VL>(p + e, w[u].n - e, v[u][r]);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float top = 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int k = 0; k < 4; k += 2) top = max_abs3(v[u][r][k], v[u][r][k + 1], top);
#pragma unroll
        for (int o = LPG / 2; o > 0; o >>= 1) top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
        const int64_t i = first + u * NG;
        if (i >= a.items) continue;
        const float s = group_scale(top), inv = group_inverse(s);
        const int width = w[u].g == a.groups - 1 ? (int)(a.ldq - (int64_t)w[u].g * a.pitch) : a.pitch;
        const int run = a.run[job];
        int8_t *q = a.q[job] ? a.q[job] + ((w[u].row * a.ldq + (int64_t)w[u].g * a.pitch) << (run > 0)) : nullptr;
        const bool keep = !ACT || q;          // an activation without a backward pass keeps nothing
        if (lane == 0 && keep) a.scale[job][i * a.scale_stride[job]] = s;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int e = (lane + r * LPG) * 4;
            if (e >= width) continue;
            if (keep)
                *reinterpret_cast<uint32_t *>(q + (run ? ((e & -run) << 1 | (e & (run - 1))) : e)) =
                    a.mode == TANGO_ROUND_NEAREST ? encode4(v[u][r], s, inv)
                                                  : encode4_mode(v[u][r], s, a.mode, a.seed, effective_call(a.call + job, a.step),
                                                                 (uint64_t)w[u].row * a.cols + (int64_t)w[u].g * a.group + e);
            if constexpr (ACT) {
                float y[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) y[k] = activate(v[u][r][k], a.act);
                store4<T, VL>(static_cast<T *>(a.y) + w[u].row * a.ldy + (int64_t)w[u].g * a.group + e, w[u].n - e, y);
            }
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
        w[u] = {0, 0, 0};
        if (i < a.items) w[u] = locate(a, i);
        s[u] = i < a.items ? __ldg(a.scale[0] + i) : 0.f;
        const int8_t *q = a.q[0] + w[u].row * a.ldq + (int64_t)w[u].g * a.pitch;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int e = (lane + r * LPG) * 4;
            word[u][r] = e < w[u].n ? __ldg(reinterpret_cast<const uint32_t *>(q + e)) : 0u;
            if constexpr (ACT)
                load4<T, VL>(static_cast<const T *>(a.x[0]) + w[u].row * a.ldx[0] + (int64_t)w[u].g * a.group + e, w[u].n - e,
                             dy[u][r]);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int e = (lane + r * LPG) * 4;
            if (e >= w[u].n) continue;
            Pair lo, hi;
            decode4(word[u][r], lo, hi);
            const float2 l = both(mul2(lo, pair(s[u], s[u]))), h = both(mul2(hi, pair(s[u], s[u])));
            float o[4] = {l.x, l.y, h.x, h.y};
            if constexpr (ACT) {
#pragma unroll
                for (int k = 0; k < 4; ++k) o[k] = __fmul_rn(dy[u][r][k], slope_of(o[k], a.act));
            }
            store4<T, VL>(static_cast<T *>(a.y) + w[u].row * a.ldy + (int64_t)w[u].g * a.group + e, w[u].n - e, o);
        }
}

template <class T, int VL, bool ACT, bool PACK>
static int launch_tile(const Rows8Args &a, int jobs, cudaStream_t st) {
    auto go = [&](auto tile, auto kernel) -> int {
        constexpr int per_block = decltype(tile)::kGroups * decltype(tile)::U;
        const int64_t blocks = ceil_div(a.items, per_block);
        if (blocks > 0x7fffffffLL) return TANGO_ESIZE;
        kernel<<<dim3((unsigned)blocks, (unsigned)jobs), kBlock, 0, st>>>(a);
        TANGO_LAUNCH_CHECK();
        return TANGO_OK;
    };
#define TANGO_ROWS8_TILE(LPG, R)                                                            \
    return PACK ? go(Tile<LPG, R>{}, rows8_pack_kernel<T, VL, LPG, R, ACT>)                 \
                : go(Tile<LPG, R>{}, rows8_unpack_kernel<T, VL, LPG, R, ACT>)
    if (a.group <= 4) TANGO_ROWS8_TILE(1, 1);
    if (a.group <= 8) TANGO_ROWS8_TILE(1, 2);
    if (a.group <= 16) TANGO_ROWS8_TILE(1, 4);
    if (a.group <= 32) TANGO_ROWS8_TILE(2, 4);
    if (a.group <= 64) TANGO_ROWS8_TILE(4, 4);
    if (a.group <= 128) TANGO_ROWS8_TILE(8, 4);
    if (a.group <= 256) TANGO_ROWS8_TILE(16, 4);
    if (a.group <= 512) TANGO_ROWS8_TILE(32, 4);
    TANGO_ROWS8_TILE(32, 8);
#undef TANGO_ROWS8_TILE
}

template <bool ACT, bool PACK>
static int launch(const Rows8Args &a, int jobs, int type, int vl, cudaStream_t st) {
#define TANGO_ROWS8_TYPE(T)                                                                                        \
    return vl == 4 ? launch_tile<T, 4, ACT, PACK>(a, jobs, st) : vl == 2 ? launch_tile<T, 2, ACT, PACK>(a, jobs, st) \
                                                                         : launch_tile<T, 1, ACT, PACK>(a, jobs, st)
    if (type == TANGO_FP32) TANGO_ROWS8_TYPE(float);
    if (type == TANGO_BF16) TANGO_ROWS8_TYPE(Bf16);
    TANGO_ROWS8_TYPE(Fp16);
#undef TANGO_ROWS8_TYPE
}

static int64_t element_bytes(int type) { return type == TANGO_FP32 ? 4 : 2; }

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
    a.wide = a.items >= 0x7fffffffLL;
    a.by_groups = fast_div(groups);
    return TANGO_OK;
}

// Elements that one access may take: what the base, the leading dimension and the first element of every group allow.
static int vector_length(const void *p, int64_t ld, int64_t rows, int64_t group, int64_t groups, int type) {
    int vl = 4;
    while (vl > 1 && (!aligned(p, vl * element_bytes(type)) || (rows > 1 && ld % vl) || (groups > 1 && group % vl))) vl /= 2;
    return vl;
}

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
    int vl = 4;
    for (int k = 0; k < n_jobs; ++k) {
        const tango_rows8_job &j = jobs[k];
        if (!j.x || !j.q || !j.scales || j.scale_stride < 1 || (rows > 1 && j.ldx < cols)) return TANGO_EINVAL;
        if (!aligned(j.x, element_bytes(type)) || !aligned(j.q, 4)) return TANGO_EALIGN;
        a.x[k] = j.x; a.ldx[k] = j.ldx; a.q[k] = j.q; a.scale[k] = j.scales;
        a.scale_stride[k] = j.scale_stride;
        a.run[k] = j.interleaved ? (int)tango_rows8_run(group) : 0;
        const int v = vector_length(j.x, j.ldx, rows, group, a.groups, type);
        if (v < vl) vl = v;
    }
    a.mode = mode; a.act = ACT_NONE; a.seed = seed; a.call = call;
    a.step = reinterpret_cast<const unsigned long long *>(step);
    return launch<false, true>(a, n_jobs, type, vl, static_cast<cudaStream_t>(stream));
}

extern "C" int tango_rows8_unpack(const int8_t *q, const float *scales, int64_t rows, int64_t cols, int64_t group, int type,
                                  void *out, int64_t ldo, tango_stream_t stream) {
    Rows8Args a{};
    const int rc = fill(a, rows, cols, group, type);
    if (rc != TANGO_OK || rows == 0 || cols == 0) return rc;
    if (!q || !scales || !out || (rows > 1 && ldo < cols)) return TANGO_EINVAL;
    if (!aligned(out, element_bytes(type)) || !aligned(q, 4)) return TANGO_EALIGN;
    a.q[0] = const_cast<int8_t *>(q); a.scale[0] = const_cast<float *>(scales); a.y = out; a.ldy = ldo; a.act = ACT_NONE;
    return launch<false, false>(a, 1, type, vector_length(out, ldo, rows, group, a.groups, type), static_cast<cudaStream_t>(stream));
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
    a.mode = mode; a.act = act; a.seed = seed; a.call = call;
    a.step = reinterpret_cast<const unsigned long long *>(step);
    const int vx = vector_length(job->x, job->ldx, rows, group, a.groups, type), vy = vector_length(y, ldy, rows, group, a.groups, type);
    return launch<true, true>(a, 1, type, vx < vy ? vx : vy, static_cast<cudaStream_t>(stream));
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
    const int vi = vector_length(dy, lddy, rows, group, a.groups, type), vo = vector_length(dx, lddx, rows, group, a.groups, type);
    return launch<true, false>(a, 1, type, vi < vo ? vi : vo, static_cast<cudaStream_t>(stream));
}
