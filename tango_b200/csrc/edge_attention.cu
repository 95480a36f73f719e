// Dot-product attention over the edges of a graph, on 8-bit rows (rows8.cuh) with one scale per node and head.
//
//   z = scale * <q[v], k[u]>,  p = softmax of z over the edges u -> v of v,  out[v] = sum p v[u]           (forward)
//   dp = <o[v], v[u]>,  delta[v] = sum p dp,  dq[v] = scale * sum p (dp - delta[v]) k[u]                    (by destination)
//   dk[u] = scale * sum p (dp - delta[v]) q[v],  dv[u] = sum p o[v]                                         (by source)
//
// where q, k, v, o (the incoming gradient) are codes times scales.  No array of edges exists: the forward pass walks a row
// once with the running maximum and sum of its softmax and leaves both per row and head; the backward passes compute the
// probabilities from them again, bit for bit (the products of codes are exact integers and the three roundings behind them
// are the same ones).  delta is not needed beforehand: dq = scale * (sum p dp k - delta sum p k), so one walk
// gathers delta and both sums, and what the forward pass has to keep is the 8-bit rows and two floats per row and head.
//
// Sums are fp32, in one order per row length and schedule (no atomics); where a few rows are asked for, per row length and number of
// blocks a row, which follows the number of rows asked for.
//
// dq as a difference of two sums leaves rounding where the formula cancels: a node with one incoming edge, whose dq is 0, gets up to
// 2^-23 |dp| |k| (dk, which knows delta beforehand, gets 0).
//
// What bounds these kernels is the gather through L1 and L2: an edge brings 2 F bytes of codes and 8 H bytes of scales (16 H by
// source), 5.8 GB for 20 M edges of 4 x 32.  On 232,965 nodes they take 529 us forward, 659 by destination and 773 by source (11.0,
// 8.8 and 8.3 TB/s of gathered bytes; 20 to 30 % of the sectors miss L2, whose near half holds no table of 60 MB), on 114.6 M edges
// of 4 x 16 1347 us forward (13.6 TB/s; on 40 M edges of the same nodes the issue slots are 70 % busy).  Without the weighted sums
// (leaving out the conversion and addition of v) the forward passes would take 527 and 1254 us where they took 615 and 1537: their
// arithmetic is mostly hidden, and matrix instructions for it would buy little.
//   * k and v (in the backward pass q and the gradient, which the pass by destination lays out for the one by source) lie in turns
//     of one lane's codes, so that a 32-byte load brings both: 20 M edges 631 -> 603 us forward, by source 913 -> 861.
//   * The loads of a lane's next edges are issued before the present ones are worked on (InFlight), and none depends on a
//     condition: slots behind a row's end read its last edge again, without weight.
//   * Codes become floats by placing the biased byte in the mantissa of 2^23, two at a time in packed fp32 arithmetic; dot products
//     of codes are exact in integers.
//   * Persistent warps that share out the short rows and fetch the next row's bounds early lost to the hardware's order of blocks
//     (603 -> 713 us at best: unequal rows), cache hints on outputs, indices and the table changed nothing.
//
// A lane holds VB neighbouring codes of one head (16, less for narrow heads), P lanes a head, L = P * (heads of a block)
// lanes an edge, and a warp as many edges side by side (slots) as fit.  None of these has to be a power of two: three heads of
// 41 are 9 lanes an edge, three edges a warp.  A long row has a warp, a short one the lanes of a slot or a few (a team); the
// longest ones are cut into units whose partial results are merged by a second launch.
#include "rows8.cuh"

namespace tango {

enum { FORWARD = 0, BY_DST = 1, BY_SRC = 2 };
constexpr int kWarps = 4, kRowWarps = 4;

// How a warp is shared out.
struct Lanes {
    int hb, l, slots;                  // heads of a block, lanes of an edge, edges side by side
    int team_slots, teams;             // slots of a short row's team, teams of a warp
    uint32_t rcp_l, rcp_team;          // 65536 / lanes, rounded up: exact quotients of the 32 lanes
};
__device__ __forceinline__ int over(int lane, uint32_t rcp) { return (int)((uint32_t)lane * rcp >> 16); }

struct AttnArgs {
    const int32_t *indptr, *indices;
    const int4 *rows, *units;                       // (row, first slot, end slot, place of a unit in its row)
    int64_t n_units, n_heavy, n_long, n_rows;       // rows: [heavy: by units] [to n_long: a warp] [the rest: a team]
    int heads, d, pitch;
    Lanes lanes;
    int ld;                                         // bytes of a row of codes
    const int8_t *q, *o, *kv;                       // kv and qo: runs of VB codes of the one and of the other in turn
    int8_t *qo;
    const float *sq, *so;                           // scales [rows, heads]
    const float2 *skv;                              // scales of k and v [rows, heads]
    float qscale;                                   // scale * log2(e)
    float2 *stats;                                  // [rows, heads]: reference of z * log2(e), 1 / sum
    float4 *record;                                 // [rows, heads], BY_DST writes and BY_SRC gathers: see there
    void *out_a, *out_b;
    int type;
    float *ws;                                      // partial results of the units
};

// Results below the normal numbers become 0: a weight that small is lost beside the row's largest, which lies between 1 and 2^kSlack.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ Pair shuffle2(Pair a, int from) { return {__shfl_sync(0xffffffffu, a.v, from)}; }

// VB codes.
template <int VB> struct Codes { uint32_t w[VB / 4]; };
template <int VB>
__device__ __forceinline__ Codes<VB> load_codes(const int8_t *p) {
    Codes<VB> c;
    if constexpr (VB == 16) {
        const uint4 t = __ldg(reinterpret_cast<const uint4 *>(p));
        c.w[0] = t.x; c.w[1] = t.y; c.w[2] = t.z; c.w[3] = t.w;
    } else if constexpr (VB == 8) {
        const uint2 t = __ldg(reinterpret_cast<const uint2 *>(p));
        c.w[0] = t.x; c.w[1] = t.y;
    } else {
        c.w[0] = __ldg(reinterpret_cast<const uint32_t *>(p));
    }
    return c;
}
// A run of one matrix and the run of the other behind it, in one access.
template <int VB>
__device__ __forceinline__ void load_runs(const int8_t *p, Codes<VB> &a, Codes<VB> &b) {
    if constexpr (VB == 16) {
        asm("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
            : "=r"(a.w[0]), "=r"(a.w[1]), "=r"(a.w[2]), "=r"(a.w[3]), "=r"(b.w[0]), "=r"(b.w[1]), "=r"(b.w[2]), "=r"(b.w[3]) : "l"(p));
    } else if constexpr (VB == 8) {
        const uint4 t = __ldg(reinterpret_cast<const uint4 *>(p));
        a.w[0] = t.x; a.w[1] = t.y; b.w[0] = t.z; b.w[1] = t.w;
    } else {
        const uint2 t = __ldg(reinterpret_cast<const uint2 *>(p));
        a.w[0] = t.x; b.w[0] = t.y;
    }
}
template <int VB>
__device__ __forceinline__ void store_runs(int8_t *p, const Codes<VB> &a, const Codes<VB> &b) {
    if constexpr (VB == 16) {
        const uint32_t w[8] = {a.w[0], a.w[1], a.w[2], a.w[3], b.w[0], b.w[1], b.w[2], b.w[3]};
        store_v8(reinterpret_cast<float *>(p), w);
    } else if constexpr (VB == 8) {
        *reinterpret_cast<uint4 *>(p) = make_uint4(a.w[0], a.w[1], b.w[0], b.w[1]);
    } else {
        *reinterpret_cast<uint2 *>(p) = make_uint2(a.w[0], b.w[0]);
    }
}
template <int VB>
__device__ __forceinline__ Codes<VB> codes_if(bool there, const int8_t *p) {
    if (there) return load_codes<VB>(p);
    Codes<VB> c;
#pragma unroll
    for (int i = 0; i < VB / 4; ++i) c.w[i] = 0;
    return c;
}
// Sum over the P lanes of a head (of which this is the one at `chunk`), the same number in all of them.
template <int P>
__device__ __forceinline__ int head_sum(int s, int lane, int chunk) {
    if constexpr ((P & (P - 1)) == 0) {             // heads start on multiples of P
#pragma unroll
        for (int o = P / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        return s;
    } else {
        int at = chunk;
        if constexpr (P == 6) {
            s += __shfl_sync(0xffffffffu, s, at < 3 ? lane + 3 : lane - 3);
            at = at < 3 ? at : at - 3;
        } else {
            static_assert(P == 3, "lanes of a head");
        }
        const int right = __shfl_sync(0xffffffffu, s, at == 2 ? lane - 2 : lane + 1);
        return s + right + __shfl_sync(0xffffffffu, s, at == 0 ? lane + 2 : lane - 1);
    }
}
// Exact product of two heads.  Up to 256 codes the sum is below 2^22 and is added up in the mantissa of 1.5 * 2^23, with which
// one lane of the head starts (`start`: dot_start).
constexpr int kMagicBits = 0x4B400000;
template <int VB, int P>
__device__ __forceinline__ int dot_start(int chunk) { return VB * P <= 256 && chunk == 0 ? kMagicBits : 0; }
template <int VB, int P>
__device__ __forceinline__ float dot(const Codes<VB> &a, const Codes<VB> &b, int start, int lane, int chunk) {
    int s = start;
#pragma unroll
    for (int i = 0; i < VB / 4; ++i) s = __dp4a((int)a.w[i], (int)b.w[i], s);
    s = head_sum<P>(s, lane, chunk);
    if constexpr (VB * P <= 256) return __fsub_rn(__int_as_float(s), kRoundMagic);
    else return __int2float_rn(s);
}
// acc += by * codes
template <int VB>
__device__ __forceinline__ void add_codes(Pair (&acc)[VB / 2], const Codes<VB> &c, Pair by) {
#pragma unroll
    for (int i = 0; i < VB / 4; ++i) {
        Pair lo, hi;
        decode4(c.w[i], lo, hi);
        acc[2 * i] = fma2(lo, by, acc[2 * i]);
        acc[2 * i + 1] = fma2(hi, by, acc[2 * i + 1]);
    }
}
// accA += a * codes, accB += b * codes
template <int VB>
__device__ __forceinline__ void add_codes_twice(Pair (&accA)[VB / 2], Pair (&accB)[VB / 2], const Codes<VB> &c, Pair a, Pair b) {
#pragma unroll
    for (int i = 0; i < VB / 4; ++i) {
        Pair lo, hi;
        decode4(c.w[i], lo, hi);
        accA[2 * i] = fma2(lo, a, accA[2 * i]);
        accA[2 * i + 1] = fma2(hi, a, accA[2 * i + 1]);
        accB[2 * i] = fma2(lo, b, accB[2 * i]);
        accB[2 * i + 1] = fma2(hi, b, accB[2 * i + 1]);
    }
}

// acc * by as elements e .. e + VB of a row of `out` (those below d).
template <class T, int VB>
__device__ __forceinline__ void store_row(T *out, int e, int d, const Pair (&acc)[VB / 2], float by) {
#pragma unroll
    for (int i = 0; i < VB; i += 4) {
        const float2 a = both(acc[i / 2]), b = both(acc[i / 2 + 1]);
        const float v[4] = {a.x * by, a.y * by, b.x * by, b.y * by};
        if (d % 4 == 0) {
            if (e + i < d) store4<T, 4>(out + e + i, 4, v);
        } else {
            store4<T, 1>(out + e + i, d - e - i, v);
        }
    }
}
template <int VB>
__device__ __forceinline__ void store_typed(void *out, int64_t at, int type, int e, int d, const Pair (&acc)[VB / 2], float by) {
    if (type == TANGO_FP32) store_row<float, VB>(static_cast<float *>(out) + at, e, d, acc, by);
    else if (type == TANGO_BF16) store_row<Bf16, VB>(static_cast<Bf16 *>(out) + at, e, d, acc, by);
    else store_row<Fp16, VB>(static_cast<Fp16 *>(out) + at, e, d, acc, by);
}
template <int VB>
__device__ __forceinline__ void store_partial(float *ws, const Pair (&acc)[VB / 2]) {
#pragma unroll
    for (int i = 0; i < VB / 2; ++i) reinterpret_cast<float2 *>(ws)[i] = both(acc[i]);
}

// Floats of a unit's partial result: per head `PartialHeads` of them, then one or two sums per code.
__host__ __device__ constexpr int partial_heads(int mode) { return mode == FORWARD ? 2 : mode == BY_DST ? 1 : 0; }
__host__ __device__ constexpr int partial_sums(int mode) { return mode == FORWARD ? 1 : 2; }
__host__ __device__ inline int64_t partial_floats(int mode, int heads, int64_t ld) {
    return (partial_heads(mode) * heads + 3) / 4 * 4 + partial_sums(mode) * ld;
}

// A softmax that is being added up: reference (of z * log2 e), sum, weighted sums of codes.  The reference follows the maximum
// only when a score passes it by kSlack: weights up to 2^kSlack are as exact in fp32 as weights up to 1, and what has been added
// up is rescaled once or twice a row, where the exact maximum changes in one of a warp's 32 softmaxes in nearly every trip
// through rows of some hundred edges.  Before the first edge the reference is the lowest number, no score but one of minus
// infinity is below it, so that nothing here has to ask for it.  A row whose scores have all passed the lowest number has the sum
// 0 and no softmax: NaN, as a row with a score above the highest number.
constexpr float kBelow = -3.402823466e38f, kSlack = 8.f;
__device__ __forceinline__ float softmax_inverse(float l, bool edges) {
    if (l == 0.f) return edges ? __int_as_float(0x7fffffff) : 0.f;
    return __fdiv_rn(1.f, l);
}
template <int VB> struct Running {
    float m = kBelow, l = 0.f;
    Pair acc[VB / 2];
    __device__ Running() {
#pragma unroll
        for (int i = 0; i < VB / 2; ++i) acc[i] = pair(0.f, 0.f);
    }
    __device__ __forceinline__ void scale(float c) {
        l *= c;
        const Pair cc = pair(c, c);
#pragma unroll
        for (int i = 0; i < VB / 2; ++i) acc[i] = mul2(acc[i], cc);
    }
    // with the same place of another slot, if there is one
    __device__ __forceinline__ void merge(int from, bool there) {
        float mo = __shfl_sync(0xffffffffu, m, from), lo = __shfl_sync(0xffffffffu, l, from);
        if (!there) { mo = kBelow; lo = 0.f; }
        const float top = fmaxf(m, mo);
        const float c = exp2_fast(m - top), co = there ? exp2_fast(mo - top) : 0.f;
        const Pair cc = pair(c, c), cco = pair(co, co);
        m = top;
        l = fmaf(l, c, lo * co);
#pragma unroll
        for (int i = 0; i < VB / 2; ++i) {
            const Pair o = shuffle2(acc[i], from);
            acc[i] = mul2(acc[i], cc);
            if (there) acc[i] = fma2(o, cco, acc[i]);
        }
    }
};

// The slots of a team meet, the lower half taking over the upper one's until the first has all: f(lane to read, whether it counts).
template <class F>
__device__ __forceinline__ void join_slots(int slots, int slot, int lane, int l, F f) {
    int o = 1;
    while (o < slots) o <<= 1;
    for (o >>= 1; o > 0; o >>= 1) {
        const bool there = slot < o && slot + o < slots;
        f(there ? lane + o * l : lane, there);
        slots = o;
    }
}

// One step of the forward pass: U edges of a lane; an edge that is not there has z = -inf and so no weight.
template <int VB, int U>
__device__ __forceinline__ void softmax_step(Running<VB> &r, const float (&z)[U], const float (&sv)[U], const Codes<VB> (&v)[U]) {
    float top = r.m;
#pragma unroll
    for (int u = 0; u < U; ++u) top = fmaxf(top, z[u]);
    const bool passed = top > r.m + kSlack;
    if (__any_sync(0xffffffffu, passed)) {
        const float to = passed ? top : r.m;
        r.scale(exp2_fast(r.m - to));
        r.m = to;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const float p = exp2_fast(z[u] - r.m);
        r.l += p;
        const float w = p * sv[u];
        add_codes<VB>(r.acc, v[u], pair(w, w));
    }
}

// Edges of a slot in one trip and blocks an SM: what is loaded one trip ahead hides the way to L2, against the registers that it
// takes.  Forward / by destination / by source, us, 20 M edges of 4 x 32: 2, 2, 2 edges with 6, 4, 4 blocks 605 / 755 / 849;
// 3, 3, 3 with 5, 3, 3 572 / 788 / 886; 4, 4, 4 with 6, 4, 4 609 / 693 / 814; as here 544 / 681 / 790 (all four on one GPU, 2 to 3 %
// slower than the one of the figures above).
template <int MODE> struct InFlight { static constexpr int U = MODE == FORWARD ? 4 : 3, kBlocks = MODE == FORWARD ? 5 : 4; };

template <int MODE, int VB, int P>
__global__ void __launch_bounds__(kWarps * 32, InFlight<MODE>::kBlocks) attn_kernel(const __grid_constant__ AttnArgs a) {
    constexpr int U = InFlight<MODE>::U;
    const int lane = threadIdx.x & 31;
    // ---- what this warp works on
    const int64_t w = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    int row = -1, beg = 0, end = 0, place = 0, slots = a.lanes.slots, in_team = lane;
    int64_t unit = -1, at = -1;
    if (w < a.n_units) {
        unit = w;
    } else {
        at = w - a.n_units + a.n_heavy;
        if (at >= a.n_long) {
            const int team = over(lane, a.lanes.rcp_team);
            slots = a.lanes.team_slots;
            in_team = lane - team * slots * a.lanes.l;
            at = team < a.lanes.teams ? a.n_long + (at - a.n_long) * a.lanes.teams + team : a.n_rows;
        }
    }
    const int L = a.lanes.l, slot = over(in_team, a.lanes.rcp_l), in_edge = in_team - slot * L;
    if (slot < slots) {                 // lanes behind the last slot have no row
        if (unit >= 0) {
            const int4 t = __ldg(a.units + unit);
            row = t.x; beg = t.y; end = t.z; place = t.w;
        } else if (at < a.n_rows) {
            if (a.rows) {
                const int4 t = __ldg(a.rows + at);
                row = t.x; beg = t.y; end = t.z;
            } else {
                row = (int)at; beg = __ldg(a.indptr + at); end = __ldg(a.indptr + at + 1);
            }
        }
    }
    const int head = blockIdx.y * a.lanes.hb + in_edge / P, chunk = in_edge % P, start = dot_start<VB, P>(chunk);
    const bool live = head < a.heads && chunk * VB < a.pitch;
    // Lanes without a place in the row read along with one that has (their own operand is 0, their results go nowhere), and
    // slots behind the row's end read its last edge once more without weight: no load and no register waits for a condition.
    const int hd = head < a.heads ? head : a.heads - 1, off = live ? head * a.pitch + chunk * VB : hd * a.pitch;

    // ---- the row's own operands
    const bool mine = row >= 0 && live;
    const int64_t rh = (int64_t)row * a.heads + hd, at_row = (int64_t)row * a.ld + off;
    Codes<VB> fa, fb;
    if constexpr (MODE == BY_SRC) {
#pragma unroll
        for (int i = 0; i < VB / 4; ++i) fa.w[i] = fb.w[i] = 0;
        if (mine) load_runs<VB>(a.kv + 2 * at_row, fa, fb);
    } else {
        fa = codes_if<VB>(mine, a.q + at_row);
        if constexpr (MODE == BY_DST) fb = codes_if<VB>(mine, a.o + at_row);
    }
    float sa = 0.f, sb = 0.f, top = 0.f, inv = 0.f;
    if (row >= 0) {
        if constexpr (MODE == BY_SRC) {
            const float2 t = __ldg(a.skv + rh);
            sa = t.x; sb = t.y;
        } else {
            sa = __ldg(a.sq + rh) * a.qscale;
        }
        if constexpr (MODE == BY_DST) {
            sb = __ldg(a.so + rh);
            const float2 st = __ldg(a.stats + rh);
            top = st.x; inv = st.y;
        }
    }
    const int8_t *base = (MODE == BY_SRC ? a.qo : a.kv) + 2 * off;
    const int ld2 = 2 * a.ld;
    const char *scales = MODE == BY_SRC ? reinterpret_cast<const char *>(a.record + hd) : reinterpret_cast<const char *>(a.skv + hd);
    const int scales_ld = a.heads * (MODE == BY_SRC ? (int)sizeof(float4) : (int)sizeof(float2));

    Running<VB> run;                    // forward: the softmax; else acc = the first sum
    Pair acc2[VB / 2];
    float delta = 0.f;
#pragma unroll
    for (int i = 0; i < VB / 2; ++i) acc2[i] = pair(0.f, 0.f);

    // One trip of a row: U edges a slot.  The next trip's loads are under way while one is worked on.
    struct Trip {
        Codes<VB> a[U], b[U];
        float2 kv[U];
        float4 rec[U];
    };
    const int stride = slots * U;
    // slots are counted without a sign: the trips ahead reach some hundred slots past a row's end, beyond 2^31 on the largest graphs
    const int trips = (int)__reduce_max_sync(0xffffffffu, ((unsigned)(end - beg) + stride - 1) / stride);
    const unsigned last = end > beg ? end - 1 : 0, behind = end;
    int next[U];
    const auto ids = [&](unsigned j) {
#pragma unroll
        for (int u = 0; u < U; ++u) next[u] = __ldg(a.indices + min(j + u * slots, last));
    };
    const auto load = [&](Trip &t) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            load_runs<VB>(base + (int64_t)next[u] * ld2, t.a[u], t.b[u]);
            const char *p = scales + (int64_t)next[u] * scales_ld;
            if constexpr (MODE == BY_SRC) t.rec[u] = __ldg(reinterpret_cast<const float4 *>(p));
            else t.kv[u] = __ldg(reinterpret_cast<const float2 *>(p));
        }
    };
    const auto work = [&](const Trip &t, unsigned j) {
        if constexpr (MODE == FORWARD) {
            float z[U], sv[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float s = dot<VB, P>(fa, t.a[u], start, lane, chunk);
                z[u] = j + u * slots < behind ? __fmul_rn(s, __fmul_rn(t.kv[u].x, sa)) : -INFINITY;
                sv[u] = t.kv[u].y;
            }
            softmax_step<VB, U>(run, z, sv, t.b);
        } else if constexpr (MODE == BY_DST) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float s = dot<VB, P>(fa, t.a[u], start, lane, chunk), dp = dot<VB, P>(fb, t.b[u], start, lane, chunk) * t.kv[u].y;
                const float z = j + u * slots < behind ? __fmul_rn(s, __fmul_rn(t.kv[u].x, sa)) : -INFINITY;
                const float p = exp2_fast(z - top) * inv;
                delta = fmaf(p, dp, delta);
                const float pk = p * t.kv[u].x, pdk = pk * dp;
                add_codes_twice<VB>(run.acc, acc2, t.a[u], pair(pdk, pdk), pair(pk, pk));
            }
        } else {
            // record of a destination: scale * log2(e) * scale of q, reference, scale of o / sum, delta / scale of o
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float s = dot<VB, P>(fa, t.a[u], start, lane, chunk), dp = dot<VB, P>(fb, t.b[u], start, lane, chunk) * sb;
                const float z = j + u * slots < behind ? __fmul_rn(s, __fmul_rn(sa, t.rec[u].x)) : -INFINITY;
                const float p = exp2_fast(z - t.rec[u].y) * t.rec[u].z;
                const float ds = p * (dp - t.rec[u].w) * t.rec[u].x;
                add_codes<VB>(run.acc, t.a[u], pair(ds, ds));
                add_codes<VB>(acc2, t.b[u], pair(p, p));
            }
        }
    };
    if (trips > 0) {
        Trip even, odd;
        unsigned j = beg + slot;
        ids(j);
        load(even);
        ids(j + stride);
        for (int t = 0;; t += 2) {
            load(odd);
            ids(j + 2 * stride);
            work(even, j);
            if (t + 1 >= trips) break;
            load(even);
            ids(j + 3 * stride);
            work(odd, j + stride);
            if (t + 2 >= trips) break;
            j += 2 * stride;
        }
    }

    join_slots(slots, slot, lane, L, [&](int from, bool there) {
        if constexpr (MODE == FORWARD) {
            run.merge(from, there);
        } else {
            const float d = __shfl_sync(0xffffffffu, delta, from);
            if (there) delta += d;
#pragma unroll
            for (int i = 0; i < VB / 2; ++i) {
                const Pair x = shuffle2(run.acc[i], from), y = shuffle2(acc2[i], from);
                if (there) {
                    run.acc[i] = add2(run.acc[i], x);
                    acc2[i] = add2(acc2[i], y);
                }
            }
        }
    });
    if (end == beg) {               // a row without edges read along with others, whose NaN is not its own
        run.l = delta = 0.f;
#pragma unroll
        for (int i = 0; i < VB / 2; ++i) run.acc[i] = acc2[i] = pair(0.f, 0.f);
    }
    if (slot != 0 || row < 0 || !live) return;
    if constexpr (MODE == BY_DST) {
        if (a.qo && place == 0) store_runs<VB>(a.qo + 2 * at_row, fa, fb);
    }
    if (unit >= 0) {
        float *ws = a.ws + unit * partial_floats(MODE, a.heads, a.ld);
        if (chunk == 0) {
            if constexpr (MODE == FORWARD) { ws[2 * head] = run.m; ws[2 * head + 1] = run.l; }
            if constexpr (MODE == BY_DST) ws[head] = delta;
        }
        ws += (partial_heads(MODE) * a.heads + 3) / 4 * 4 + off;
        store_partial<VB>(ws, run.acc);
        if constexpr (MODE != FORWARD) store_partial<VB>(ws + a.ld, acc2);
        return;
    }
    const int64_t out = rh * a.d;
    const int e = chunk * VB;
    if constexpr (MODE == FORWARD) {
        const float by = softmax_inverse(run.l, end > beg);
        store_typed<VB>(a.out_a, out, a.type, e, a.d, run.acc, by);
        if (chunk == 0 && a.stats) a.stats[rh] = make_float2(run.l == 0.f ? 0.f : run.m, by);
    } else if constexpr (MODE == BY_DST) {
        const Pair nd = pair(-delta, -delta);
#pragma unroll
        for (int i = 0; i < VB / 2; ++i) run.acc[i] = fma2(acc2[i], nd, run.acc[i]);
        store_typed<VB>(a.out_a, out, a.type, e, a.d, run.acc, a.qscale * 0.69314718055994531f * sb);
        if (chunk == 0 && a.record) a.record[rh] = make_float4(sa, top, inv * sb, delta);
    } else {
        store_typed<VB>(a.out_a, out, a.type, e, a.d, run.acc, 0.69314718055994531f);
        store_typed<VB>(a.out_b, out, a.type, e, a.d, acc2, 1.f);
    }
}

// A block per heavy row.  Its threads stand for the codes of a row, several times over: each takes every G-th unit, and the G
// partial results meet in shared memory.
struct MergeArgs {
    const int4 *rows;
    const int32_t *heavy_first;
    int heads, d, pitch, ld;
    const float *ws;
    const float *sq, *so;
    float qscale;
    float2 *stats;
    float4 *record;
    void *out_a, *out_b;
    int type;
};
__device__ __forceinline__ void store_one(void *out, int64_t at, int type, float v) {
    if (type == TANGO_FP32) static_cast<float *>(out)[at] = v;
    else if (type == TANGO_BF16) from_float(v, static_cast<Bf16 *>(out)[at]);
    else from_float(v, static_cast<Fp16 *>(out)[at]);
}
constexpr int kMergeThreads = 512;

template <int MODE>
__global__ void __launch_bounds__(kMergeThreads) attn_merge_kernel(const __grid_constant__ MergeArgs a) {
    __shared__ float s_x[kMergeThreads], s_y[kMergeThreads], s_z[kMergeThreads];
    const int4 heavy = __ldg(a.rows + blockIdx.x);
    const int64_t row = heavy.x;
    const int first = __ldg(a.heavy_first + blockIdx.x), n = __ldg(a.heavy_first + blockIdx.x + 1) - first;
    const int64_t step = partial_floats(MODE, a.heads, a.ld);
    const float *ws = a.ws + (int64_t)first * step;
    const int per_head = (partial_heads(MODE) * a.heads + 3) / 4 * 4;
    const int width = a.ld < kMergeThreads ? a.ld : kMergeThreads, G = kMergeThreads / width;
    const int g = threadIdx.x / width, in = threadIdx.x % width;
    for (int e0 = 0; e0 < a.ld; e0 += width) {
        const int e = e0 + in, head = e / a.pitch, i = e - head * a.pitch;
        const bool there = g < G && e < a.ld;
        // forward: x sum, y maximum, z sum of weights; by destination: both sums and delta; by source: both sums
        float x = 0.f, y = MODE == FORWARD ? kBelow : 0.f, z = 0.f;
        if (there) {
            if constexpr (MODE == FORWARD) {
#pragma unroll 4
                for (int u = g; u < n; u += G) y = fmaxf(y, ws[u * step + 2 * head]);
            }
#pragma unroll 4
            for (int u = g; u < n; u += G) {
                const float *p = ws + u * step;
                if constexpr (MODE == FORWARD) {
                    const float c = exp2_fast(p[2 * head] - y);
                    z = fmaf(p[2 * head + 1], c, z);
                    x = fmaf(p[per_head + e], c, x);
                } else {
                    if constexpr (MODE == BY_DST) z += p[head];
                    x += p[per_head + e];
                    y += p[per_head + a.ld + e];
                }
            }
        }
        s_x[threadIdx.x] = x; s_y[threadIdx.x] = y; s_z[threadIdx.x] = z;
        __syncthreads();
        if (g == 0 && there && i < a.d) {
            const int64_t rh = row * a.heads + head, out = rh * a.d + i;
            float m = y;
            if constexpr (MODE == FORWARD) {
                for (int k = 1; k < G; ++k) m = fmaxf(m, s_y[k * width + in]);
                const float c = exp2_fast(y - m);
                x *= c; z *= c;
            }
            for (int k = 1; k < G; ++k) {
                const int at = k * width + in;
                if constexpr (MODE == FORWARD) {
                    const float c = exp2_fast(s_y[at] - m);
                    x = fmaf(s_x[at], c, x);
                    z = fmaf(s_z[at], c, z);
                } else {
                    x += s_x[at]; y += s_y[at]; z += s_z[at];
                }
            }
            if constexpr (MODE == FORWARD) {
                const float by = softmax_inverse(z, heavy.z > heavy.y);
                store_one(a.out_a, out, a.type, x * by);
                if (i == 0 && a.stats) a.stats[rh] = make_float2(z == 0.f ? 0.f : m, by);
            } else if constexpr (MODE == BY_DST) {
                const float sb = a.so[rh];
                store_one(a.out_a, out, a.type, fmaf(y, -z, x) * (a.qscale * 0.69314718055994531f * sb));
                if (i == 0 && a.record) {
                    const float2 st = a.stats[rh];
                    a.record[rh] = make_float4(a.sq[rh] * a.qscale, st.x, st.y * sb, z);
                }
            } else {
                store_one(a.out_a, out, a.type, x * 0.69314718055994531f);
                store_one(a.out_b, out, a.type, y);
            }
        }
        __syncthreads();
    }
}

// ---- a few rows whose queries just arrived: a whole block a row, long rows over several blocks
struct RowsArgs {
    const int32_t *indptr, *indices;
    const int64_t *rows;
    int64_t n_nodes;
    const void *q;
    int64_t ldq;                  // elements between two queries
    int heads, d, pitch;
    Lanes lanes;
    int ld;
    const int8_t *k, *v;
    const float *sk, *sv;
    float qscale;
    int splits;                   // blocks a row may be cut into
    void *out;
    int type;
    float *ws;                    // [rows, splits] partial results
    int mode;
    uint64_t seed, call;
    const unsigned long long *step;
};
constexpr int kRowChunk = 256;    // edges below which a row is not cut: four trips of a block of F = 128

__host__ __device__ inline int row_chunk(int len, int splits) {
    const int c = (int)(((unsigned)len + splits - 1) / splits);
    return c < kRowChunk ? kRowChunk : c;
}

template <int VB, class T>
__device__ __forceinline__ void load_query(const RowsArgs &a, int64_t r, int head, int chunk, bool live, float (&v)[VB]) {
    const T *p = static_cast<const T *>(a.q) + r * a.ldq + (int64_t)head * a.d + chunk * VB;
#pragma unroll
    for (int i = 0; i < VB; i += 4) load4<T, 1>(p + i, live ? min(4, a.d - chunk * VB - i) : 0, v + i);
}
template <int VB, int P>
__device__ __forceinline__ Codes<VB> encode_query(const RowsArgs &a, int64_t r, int head, int chunk, const float (&v)[VB], float &s) {
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < VB; k += 2) top = max_abs3(v[k], v[k + 1], top);
    const int lane = threadIdx.x & 31, first = lane - chunk;
    float all = top;
#pragma unroll
    for (int k = 0; k < P; ++k) all = max_or_nan(all, __shfl_sync(0xffffffffu, top, first + k));
    top = all;
    s = group_scale(top);
    Codes<VB> c;
    if (a.mode == TANGO_ROUND_NEAREST) {
        encode_nearest<VB / 4>(v, s, group_inverse(s), c.w);
    } else {
#pragma unroll
        for (int i = 0; i < VB / 4; ++i)
            c.w[i] = encode4_mode(four(v + 4 * i), s, a.mode, a.seed, effective_call(a.call, a.step),
                                  (uint64_t)r * a.heads * a.d + head * a.d + chunk * VB + 4 * i);
    }
    return c;
}

template <int VB, int P>
__global__ void __launch_bounds__(kRowWarps * 32, 5) attn_rows_kernel(const __grid_constant__ RowsArgs a) {
    constexpr int U = 4;
    __shared__ float s_acc[kRowWarps][32 * VB];
    __shared__ float2 s_ml[kRowWarps][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t r = blockIdx.x;
    const int64_t row = __ldg(a.rows + r);
    const int L = a.lanes.l, slots = a.lanes.slots;
    const int slot = over(lane, a.lanes.rcp_l), in_edge = lane - slot * L;
    const int head = blockIdx.z * a.lanes.hb + in_edge / P, chunk = in_edge % P, start = dot_start<VB, P>(chunk);
    const bool live = head < a.heads && chunk * VB < a.pitch, counts = slot < slots;      // lanes behind the last slot do not count
    const int hd = head < a.heads ? head : a.heads - 1, off = live ? head * a.pitch + chunk * VB : hd * a.pitch;
    // A short row is a chain of loads (bounds, ids, keys and values) that the query's does not depend on: it is asked for first
    // and rounded while the first keys are on their way.
    float query[VB];
    if (a.type == TANGO_FP32) load_query<VB, float>(a, r, head, chunk, live, query);
    else if (a.type == TANGO_BF16) load_query<VB, Bf16>(a, r, head, chunk, live, query);
    else load_query<VB, Fp16>(a, r, head, chunk, live, query);
    const bool known = row >= 0 && row < a.n_nodes;
    const int beg0 = known ? __ldg(a.indptr + row) : 0, end0 = known ? __ldg(a.indptr + row + 1) : 0;
    const int chunk_len = row_chunk(end0 - beg0, a.splits);
    const bool whole = end0 - beg0 <= chunk_len;
    if (blockIdx.y > 0 && (int64_t)blockIdx.y * chunk_len >= end0 - beg0) return;
    const int beg = beg0 + blockIdx.y * chunk_len, end = end0 - beg < chunk_len ? end0 : beg + chunk_len;

    Running<VB> run;
    const int stride = slots * U * kRowWarps;
    unsigned j = beg + warp * slots * U;            // without a sign, as in attn_kernel
    const unsigned behind = end;
    int at[U];
    Codes<VB> ga[U], gb[U];
    float sk[U], sv[U];
    const auto ids = [&](unsigned j) {
#pragma unroll
        for (int u = 0; u < U; ++u) at[u] = __ldg(a.indices + min(j + u * slots + slot, behind - 1));
    };
    const auto load = [&] {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            ga[u] = load_codes<VB>(a.k + (int64_t)at[u] * a.ld + off);
            gb[u] = load_codes<VB>(a.v + (int64_t)at[u] * a.ld + off);
            sk[u] = __ldg(a.sk + (int64_t)at[u] * a.heads + hd);
            sv[u] = __ldg(a.sv + (int64_t)at[u] * a.heads + hd);
        }
    };
    if (j < behind) {
        ids(j);
        load();
        ids(j + stride);
    }
    float sa;
    const Codes<VB> fa = encode_query<VB, P>(a, r, head, chunk, query, sa);
    sa *= a.qscale;
    while (j < behind) {
        float z[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float s = dot<VB, P>(fa, ga[u], start, lane, chunk);
            z[u] = counts && j + u * slots + slot < behind ? __fmul_rn(s, __fmul_rn(sk[u], sa)) : -INFINITY;
        }
        softmax_step<VB, U>(run, z, sv, gb);
        j += stride;
        if (j >= behind) break;
        load();
        ids(j + stride);
    }
    join_slots(slots, slot, lane, L, [&](int from, bool there) { run.merge(from, there); });
    if (slot == 0) {
        s_ml[warp][in_edge] = make_float2(run.m, run.l);
#pragma unroll
        for (int i = 0; i < VB / 2; ++i) reinterpret_cast<float2 *>(s_acc[warp])[in_edge * (VB / 2) + i] = both(run.acc[i]);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < L * VB; e += kRowWarps * 32) {
        const int ie = e / VB, hd = blockIdx.z * a.lanes.hb + ie / P, i = ie % P * VB + e % VB;
        if (hd >= a.heads || i >= a.d) continue;
        float m = kBelow, l = 0.f, s = 0.f;
#pragma unroll
        for (int w = 0; w < kRowWarps; ++w) m = fmaxf(m, s_ml[w][ie].x);
#pragma unroll
        for (int w = 0; w < kRowWarps; ++w) {
            const float2 ml = s_ml[w][ie];
            const float c = exp2_fast(ml.x - m);
            l = fmaf(ml.y, c, l);
            s = fmaf(s_acc[w][e], c, s);
        }
        if (whole) {
            const float by = known ? softmax_inverse(l, end0 > beg0) : __int_as_float(0x7fffffff);
            store_one(a.out, (r * a.heads + hd) * a.d + i, a.type, s * by);
        } else {
            float *ws = a.ws + (r * a.splits + blockIdx.y) * partial_floats(FORWARD, a.heads, a.ld);
            if (i == 0) { ws[2 * hd] = m; ws[2 * hd + 1] = l; }
            ws[(2 * a.heads + 3) / 4 * 4 + hd * a.pitch + i] = s;
        }
    }
}

__global__ void __launch_bounds__(256) attn_rows_merge_kernel(const __grid_constant__ RowsArgs a) {
    const int64_t r = blockIdx.x, row = __ldg(a.rows + r);
    if (row < 0 || row >= a.n_nodes) return;
    const int len = __ldg(a.indptr + row + 1) - __ldg(a.indptr + row), chunk_len = row_chunk(len, a.splits);
    if (len <= chunk_len) return;
    const int n = (int)(((unsigned)len + chunk_len - 1) / chunk_len), per_head = (2 * a.heads + 3) / 4 * 4;
    const int64_t step = partial_floats(FORWARD, a.heads, a.ld);
    const float *ws = a.ws + r * a.splits * step;
    for (int e = threadIdx.x; e < a.ld; e += blockDim.x) {
        const int head = e / a.pitch, i = e - head * a.pitch;
        if (i >= a.d) continue;
        float m = kBelow, l = 0.f, s = 0.f;
        for (int u = 0; u < n; ++u) m = fmaxf(m, ws[u * step + 2 * head]);
        for (int u = 0; u < n; ++u) {
            const float c = exp2_fast(ws[u * step + 2 * head] - m);
            l = fmaf(ws[u * step + 2 * head + 1], c, l);
            s = fmaf(ws[u * step + per_head + e], c, s);
        }
        store_one(a.out, (r * a.heads + head) * a.d + i, a.type, s * softmax_inverse(l, true));
    }
}

// ---- host side
constexpr int kMaxHeadWidth = 512;

// The instantiation of a head width: codes of a lane and lanes of a head.
template <class F>
static int with_shape(int d, F f) {
    if (d <= 4) return f(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{});
    if (d <= 8) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
    const std::integral_constant<int, 16> vb{};
    if (d <= 16) return f(vb, std::integral_constant<int, 1>{});
    if (d <= 32) return f(vb, std::integral_constant<int, 2>{});
    if (d <= 48) return f(vb, std::integral_constant<int, 3>{});
    if (d <= 64) return f(vb, std::integral_constant<int, 4>{});
    if (d <= 96) return f(vb, std::integral_constant<int, 6>{});
    if (d <= 128) return f(vb, std::integral_constant<int, 8>{});
    if (d <= 256) return f(vb, std::integral_constant<int, 16>{});
    return f(vb, std::integral_constant<int, 32>{});
}
// Heads of a block: as many as fit, unless fewer leave clearly fewer lanes idle.  (A head's lanes all have work, so that idle ones
// are those behind the last slot and those of heads that a last block lacks.)
static Lanes share_out(int heads, int p) {
    Lanes best{};
    double most = 0;
    for (int hb = heads < 32 / p ? heads : 32 / p; hb >= 1; --hb) {
        const int l = hb * p, slots = 32 / l, blocks = (heads + hb - 1) / hb;
        const double busy = (double)heads / (blocks * hb) * (slots * l) / 32;
        if (busy <= most * 1.1) continue;
        most = busy;
        // a short row's team: about eight lanes
        const int team_slots = l < 8 ? 8 / l : 1;
        best = {hb, l, slots, team_slots, 32 / (team_slots * l), (uint32_t)(65536 + l - 1) / l,
                (uint32_t)(65536 + team_slots * l - 1) / (team_slots * l)};
    }
    return best;
}
static bool known_type(int type) { return type >= TANGO_FP32 && type <= TANGO_FP16; }

static int check_shape(int64_t n_rows, int heads, int d, int type) {
    if (n_rows < 0 || heads < 1 || d < 1 || !known_type(type)) return TANGO_EINVAL;
    if (d > kMaxHeadWidth || heads > 65535 || n_rows > 0x7fffffffLL) return TANGO_ESIZE;
    return TANGO_OK;
}

template <int MODE>
static int launch(AttnArgs a, const tango_edge_plan *plan, float *ws, int64_t ws_bytes, cudaStream_t st) {
    a.n_long = a.n_rows;
    if (plan) {
        a.rows = reinterpret_cast<const int4 *>(plan->rows);
        a.units = reinterpret_cast<const int4 *>(plan->units);
        a.n_units = plan->n_units; a.n_heavy = plan->n_heavy; a.n_long = plan->n_long;
        if (!plan->rows || a.n_heavy < 0 || a.n_units < a.n_heavy || a.n_long < a.n_heavy || a.n_long > a.n_rows) return TANGO_EINVAL;
        if (a.n_heavy == 0 && a.n_units > 0) return TANGO_EINVAL;
        if (a.n_heavy > 0 && (!plan->units || !plan->heavy_first || !ws || ws_bytes < a.n_units * partial_floats(MODE, a.heads, a.ld) * 4))
            return TANGO_EINVAL;
        if (!aligned(plan->rows, 16) || !aligned(plan->units, 16) || !aligned(ws, 16)) return TANGO_EALIGN;
    }
    a.ws = ws;
    const int rc = with_shape(a.d, [&](auto vb, auto p) -> int {
        constexpr int VB = decltype(vb)::value, P = decltype(p)::value;
        a.lanes = share_out(a.heads, P);
        const int64_t warps = a.n_units + (a.n_long - a.n_heavy) + ceil_div(a.n_rows - a.n_long, a.lanes.teams);
        const int64_t blocks = ceil_div(warps, kWarps), by = ceil_div(a.heads, a.lanes.hb);
        if (blocks > 0x7fffffffLL || by > 65535) return TANGO_ESIZE;
        attn_kernel<MODE, VB, P><<<dim3((unsigned)blocks, (unsigned)by), kWarps * 32, 0, st>>>(a);
        TANGO_LAUNCH_CHECK();
        return TANGO_OK;
    });
    if (rc != TANGO_OK || a.n_heavy == 0) return rc;
    MergeArgs m{a.rows, plan->heavy_first, a.heads, a.d, a.pitch, a.ld, ws, a.sq, a.so, a.qscale,
                a.stats, a.record, a.out_a, a.out_b, a.type};
    attn_merge_kernel<MODE><<<(unsigned)a.n_heavy, kMergeThreads, 0, st>>>(m);
    TANGO_LAUNCH_CHECK();
    return TANGO_OK;
}

static bool good_codes(const int8_t *q, int d) { return q && aligned(q, d > 8 ? 16 : d > 4 ? 8 : 4); }

// The 8-bit operands of a pass; the gradient's belong to the backward pass.
static int operands(AttnArgs &a, const tango_edge_operands *x, bool backward) {
    if (!x || !good_codes(x->q, a.d) || !x->kv || !x->sq || !x->skv) return TANGO_EINVAL;
    if (backward && (!good_codes(x->o, a.d) || !x->so)) return TANGO_EINVAL;
    if (!aligned(x->skv, 8) || !aligned(x->kv, 32)) return TANGO_EALIGN;
    a.q = x->q; a.kv = x->kv; a.o = x->o; a.sq = x->sq; a.so = x->so;
    a.skv = reinterpret_cast<const float2 *>(x->skv);
    return TANGO_OK;
}

static AttnArgs attn_args(const int32_t *indptr, const int32_t *indices, int64_t n_rows, int heads, int d, float scale, int type) {
    AttnArgs a{};
    a.indptr = indptr; a.indices = indices; a.n_rows = n_rows;
    a.heads = heads; a.d = d; a.pitch = (int)tango_rows8_pitch(d); a.ld = heads * a.pitch;
    a.qscale = scale * 1.4426950408889634f;
    a.type = type;
    return a;
}

}  // namespace tango

using namespace tango;

extern "C" int64_t tango_edge_attention_workspace_bytes(int pass, int64_t n_units, int heads, int d) {
    if (pass < FORWARD || pass > BY_SRC || n_units < 0 || heads < 1 || d < 1) return TANGO_EINVAL;
    if (d > kMaxHeadWidth || heads > 65535 || n_units > (1LL << 31)) return TANGO_ESIZE;
    return n_units * partial_floats(pass, heads, heads * tango_rows8_pitch(d)) * 4;
}

extern "C" int tango_edge_attention(const int32_t *indptr, const int32_t *indices, int64_t n_rows, const tango_edge_plan *plan,
                                    int heads, int d, const tango_edge_operands *x, float scale, void *out, int type, float *stats,
                                    void *ws, int64_t ws_bytes, tango_stream_t stream) {
    const int rc = check_shape(n_rows, heads, d, type);
    if (rc != TANGO_OK || n_rows == 0) return rc;
    if (!indptr || !indices || !out) return TANGO_EINVAL;
    AttnArgs a = attn_args(indptr, indices, n_rows, heads, d, scale, type);
    if (const int bad = operands(a, x, false)) return bad;
    if (!aligned(out, 16) || !aligned(stats, 8)) return TANGO_EALIGN;
    a.stats = reinterpret_cast<float2 *>(stats); a.out_a = out;
    return launch<FORWARD>(a, plan, static_cast<float *>(ws), ws_bytes, static_cast<cudaStream_t>(stream));
}

extern "C" int tango_edge_attention_bwd_dst(const int32_t *indptr, const int32_t *indices, int64_t n_rows, const tango_edge_plan *plan,
                                            int heads, int d, const tango_edge_operands *x, float scale, const float *stats, void *dq,
                                            int type, float *record, int8_t *qo, void *ws, int64_t ws_bytes, tango_stream_t stream) {
    const int rc = check_shape(n_rows, heads, d, type);
    if (rc != TANGO_OK || n_rows == 0) return rc;
    if (!indptr || !indices || !dq || !stats || !record != !qo) return TANGO_EINVAL;
    AttnArgs a = attn_args(indptr, indices, n_rows, heads, d, scale, type);
    if (const int bad = operands(a, x, true)) return bad;
    if (!aligned(dq, 16) || !aligned(stats, 8) || !aligned(record, 16) || !aligned(qo, 32)) return TANGO_EALIGN;
    a.stats = reinterpret_cast<float2 *>(const_cast<float *>(stats)); a.record = reinterpret_cast<float4 *>(record); a.out_a = dq; a.qo = qo;
    return launch<BY_DST>(a, plan, static_cast<float *>(ws), ws_bytes, static_cast<cudaStream_t>(stream));
}

extern "C" int tango_edge_attention_bwd_src(const int32_t *indptr, const int32_t *indices, int64_t n_rows, const tango_edge_plan *plan,
                                            int heads, int d, const int8_t *kv, const float *skv, const int8_t *qo, const float *record,
                                            void *dk, void *dv, int type, void *ws, int64_t ws_bytes, tango_stream_t stream) {
    const int rc = check_shape(n_rows, heads, d, type);
    if (rc != TANGO_OK || n_rows == 0) return rc;
    if (!indptr || !indices || !dk || !dv || !kv || !skv || !qo || !record) return TANGO_EINVAL;
    if (!aligned(dk, 16) || !aligned(dv, 16) || !aligned(record, 16) || !aligned(kv, 32) || !aligned(qo, 32) || !aligned(skv, 8))
        return TANGO_EALIGN;
    AttnArgs a = attn_args(indptr, indices, n_rows, heads, d, 0.f, type);
    a.kv = kv; a.skv = reinterpret_cast<const float2 *>(skv); a.qo = const_cast<int8_t *>(qo);
    a.record = reinterpret_cast<float4 *>(const_cast<float *>(record)); a.out_a = dk; a.out_b = dv;
    return launch<BY_SRC>(a, plan, static_cast<float *>(ws), ws_bytes, static_cast<cudaStream_t>(stream));
}

extern "C" int tango_edge_attention_rows_splits(int64_t n_rows, int64_t longest) {
    if (n_rows < 0 || longest < 0) return TANGO_EINVAL;
    if (n_rows == 0 || longest <= kRowChunk) return 1;
    // Most of a row's blocks find nothing to do unless it is a long one, and take their turn all the same: 1024 rows of 20 M
    // edges (62 in the middle, 2021 at most), 4 x 32, take 39 us with one block a row, 26 with 4, 28 with 8 (from HBM).  From 2049
    // rows on a row is one block's, however long it is.
    const int64_t want = ceil_div(longest, kRowChunk), most = 4096 / n_rows < 64 ? 4096 / n_rows : 64;
    return (int)(want < most ? want : most < 1 ? 1 : most);
}

extern "C" int64_t tango_edge_attention_rows_workspace_bytes(int64_t n_rows, int splits, int heads, int d) {
    if (n_rows < 0 || splits < 1 || heads < 1 || d < 1) return TANGO_EINVAL;
    if (d > kMaxHeadWidth || heads > 65535 || splits > 65535 || n_rows > 0x7fffffffLL) return TANGO_ESIZE;
    return splits == 1 ? 0 : n_rows * splits * partial_floats(FORWARD, heads, heads * tango_rows8_pitch(d)) * 4;
}

extern "C" int tango_edge_attention_rows(const int32_t *indptr, const int32_t *indices, int64_t n_nodes, const int64_t *rows,
                                         int64_t n_rows, int splits, int heads, int d, const void *q, int64_t ldq, int type,
                                         const tango_rows8 *k, const tango_rows8 *v, float scale, void *out, void *ws,
                                         int64_t ws_bytes, int mode, uint64_t seed, uint64_t call, const uint64_t *step,
                                         tango_stream_t stream) {
    const int rc = check_shape(n_rows, heads, d, type);
    if (rc != TANGO_OK) return rc;
    if (n_nodes < 0 || splits < 1 || mode < TANGO_ROUND_TRUNC || mode > TANGO_ROUND_STOCHASTIC) return TANGO_EINVAL;
    if (splits > 65535) return TANGO_ESIZE;
    if (n_rows == 0) return TANGO_OK;
    if (!indptr || !indices || !rows || !q || !out || (n_rows > 1 && ldq < (int64_t)heads * d)) return TANGO_EINVAL;
    if (n_nodes > 0 && (!k || !v || !good_codes(k->q, d) || !good_codes(v->q, d) || !k->scales || !v->scales)) return TANGO_EINVAL;
    if (splits > 1 && (!ws || ws_bytes < tango_edge_attention_rows_workspace_bytes(n_rows, splits, heads, d))) return TANGO_EINVAL;
    const int element = type == TANGO_FP32 ? 4 : 2;
    if (!aligned(q, element) || !aligned(out, element) || !aligned(ws, 16)) return TANGO_EALIGN;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    RowsArgs a{};
    a.indptr = indptr; a.indices = indices; a.rows = rows; a.n_nodes = n_nodes; a.q = q; a.ldq = ldq;
    a.heads = heads; a.d = d; a.pitch = (int)tango_rows8_pitch(d); a.ld = heads * a.pitch;
    if (n_nodes > 0) { a.k = k->q; a.sk = k->scales; a.v = v->q; a.sv = v->scales; }
    a.qscale = scale * 1.4426950408889634f; a.splits = splits; a.out = out; a.type = type; a.ws = static_cast<float *>(ws);
    a.mode = mode; a.seed = seed; a.call = call; a.step = reinterpret_cast<const unsigned long long *>(step);
    const int done = with_shape(d, [&](auto vb, auto p) -> int {
        constexpr int VB = decltype(vb)::value, P = decltype(p)::value;
        a.lanes = share_out(heads, P);
        const int64_t bz = ceil_div(heads, a.lanes.hb);
        if (bz > 65535) return TANGO_ESIZE;
        attn_rows_kernel<VB, P><<<dim3((unsigned)n_rows, (unsigned)splits, (unsigned)bz), kRowWarps * 32, 0, st>>>(a);
        TANGO_LAUNCH_CHECK();
        return TANGO_OK;
    });
    if (done != TANGO_OK || splits == 1) return done;
    attn_rows_merge_kernel<<<(unsigned)n_rows, 256, 0, st>>>(a);
    TANGO_LAUNCH_CHECK();
    return TANGO_OK;
}
