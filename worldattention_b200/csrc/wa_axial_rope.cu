// Rotary embedding of tokens that each have a position of their own on several axes (time, height, width).
//
//     (a, b) -> (a cos - b sin, a sin + b cos),     cos, sin = table[positions[token, axis of the pair], pair]
//
// wa_qk_norm_rope (causal_rope_apply, wan/modules/causal_model.py:34-62) lays all samples of a batch out on one grid; here samples
// of different grids, text between pictures and single tokens share a call.  The gradient is the same turn with -sin.
// Arithmetic in float32, one rounding at the end.
//
// Bound: HBM, each value read once and written once.  A warp takes 2 KB of a token: its loads leave first, then the lanes look the cosines and sines
// of their pairs up (from L2, or from what a warp beside fetched for other heads of the token).
// 32 766 tokens of 20 heads of 128 channels: float32 103 us (6.5 TB/s, a copy's rate), bf16 61 (neighbouring pairs) and 66 (halves), where instructions and the
// registers of a lane's eight angles count, too: four thread blocks to an SM (packed multiply-adds 67, five thread blocks 78).
#include "wa_common.cuh"

namespace wa {

constexpr int AR_TENSORS = 4, AR_AXES = 8, AR_WARPS = 8;

struct AxialRope {
    View4 x[AR_TENSORS];
    void *out[AR_TENSORS];
    long long ob[AR_TENSORS], ol[AR_TENSORS], oh[AR_TENSORS];
    int heads[AR_TENSORS];
    int tensors, D, pairs, axes, rows;
    int end[AR_AXES];                 // first pair behind each axis
    long long tokens;                 // of the batch
    int L;
    const int32_t *positions;
    long long psb, psl;               // elements between samples (0: the same for all) and between tokens
    const float2 *table;              // [rows, pairs] (cos, sin)
    float sign;                       // of the angle
    int wide;                         // two neighbouring pairs of a row are 16 bytes: an even number of pairs, an aligned table
    int groups_of[AR_TENSORS];        // vector form: head groups of each tensor
};

constexpr int ar_groups(bool interleaved) { return interleaved ? 4 : 2; }        // head groups of a warp: four vectors of a lane

// cos and sin of a pair; a position outside the table gives NaN, so that it shows in the result instead of some row's angle
__device__ __forceinline__ float2 ar_turn(const AxialRope &p, const int32_t *pos, int pair) {
    int axis = 0;
#pragma unroll
    for (int a = 0; a < AR_AXES - 1; ++a) axis += a < p.axes - 1 && pair >= p.end[a];
    const int row = __ldg(pos + axis);
    if ((unsigned)row >= (unsigned)p.rows) return make_float2(NAN, NAN);
    const float2 t = __ldg(p.table + (long long)row * p.pairs + pair);
    return make_float2(t.x, t.y * p.sign);
}

// the same for `N` consecutive pairs; they mostly are of one axis or two (behind the last pair: no turn)
template <int N>
__device__ __forceinline__ void ar_turns(const AxialRope &p, const int32_t *pos, int first, float2 (&turn)[N]) {
    const int last = min(first + N, p.pairs) - 1;
    int a0 = 0, a1 = 0;
#pragma unroll
    for (int a = 0; a < AR_AXES - 1; ++a)
        if (a < p.axes - 1) {
            a0 += first >= p.end[a];
            a1 += last >= p.end[a];
        }
    if (first <= last && a1 - a0 <= 1) {
        const int r0 = __ldg(pos + a0), r1 = __ldg(pos + a1), border = p.end[a0];
        const bool in0 = (unsigned)r0 < (unsigned)p.rows, in1 = (unsigned)r1 < (unsigned)p.rows;
        const float2 *t0 = p.table + (long long)(in0 ? r0 : 0) * p.pairs + first, *t1 = p.table + (long long)(in1 ? r1 : 0) * p.pairs + first;
        if (p.wide) {          // two pairs a load; the second of two may be another axis'
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                const bool one = first + i < border, next = first + i + 1 < border;
                float4 t = make_float4(1.f, 0.f, 1.f, 0.f);
                if (first + i <= last) t = __ldg(reinterpret_cast<const float4 *>((one ? t0 : t1) + i));
                if (one && !next) {
                    const float2 u = __ldg(t1 + i + 1);
                    t.z = u.x;
                    t.w = u.y;
                }
                turn[i] = (one ? in0 : in1) ? make_float2(t.x, t.y * p.sign) : make_float2(NAN, NAN);
                turn[i + 1] = (next ? in0 : in1) ? make_float2(t.z, t.w * p.sign) : make_float2(NAN, NAN);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const bool one = first + i < border;
                turn[i] = make_float2(1.f, 0.f);
                if (first + i <= last) turn[i] = __ldg((one ? t0 : t1) + i);
                turn[i].y *= p.sign;
                if (!(one ? in0 : in1) && first + i <= last) turn[i] = make_float2(NAN, NAN);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) turn[i] = first + i <= last ? ar_turn(p, pos, first + i) : make_float2(1.f, 0.f);
    }
}

template <typename T> struct ArVec;
template <> struct ArVec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void get(uint4 w, float (&f)[8]) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(u[i] << 16), f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
    static __device__ __forceinline__ uint4 put(const float (&f)[8]) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            u[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        return make_uint4(u[0], u[1], u[2], u[3]);
    }
};
template <> struct ArVec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void get(uint4 w, float (&f)[4]) {
        f[0] = __uint_as_float(w.x), f[1] = __uint_as_float(w.y), f[2] = __uint_as_float(w.z), f[3] = __uint_as_float(w.w);
    }
    static __device__ __forceinline__ uint4 put(const float (&f)[4]) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
};

// `INTER`: a pair is two neighbouring channels, and a lane's vector holds whole pairs.  Otherwise a pair is channels i and i + pairs,
// and a lane takes the two vectors that hold its pairs' halves.  Channels behind the turned ones are copied.
// `ALL`: of neighbouring pairs every one is turned, none has to be looked at (24 heads of 4680 tokens 12.6 -> 12.0 us).
template <typename T, bool INTER, bool ALL>
__global__ void __launch_bounds__(AR_WARPS * 32)
axial_rope_vec_kernel(const __grid_constant__ AxialRope p) {
    using V = ArVec<T>;
    constexpr int N = V::N, TURNS = INTER ? N / 2 : N, AT_ONCE = ar_groups(INTER);
    pdl_wait();
    // (no division: the samples are the grid's z, the parts of a token its y)
    const int l = blockIdx.x * AR_WARPS + (threadIdx.x >> 5), b = blockIdx.z, part = blockIdx.y;
    if (l >= p.L) return;
    const int lane = threadIdx.x & 31;
    const int per_head = (INTER ? p.D : p.pairs) / N, at_once = 32 / per_head;      // lanes a head takes, heads a group holds
    const int sub = lane / per_head, c = lane - sub * per_head;                     // head within the group, vector within the head
    const T *src[AT_ONCE];
    T *dst[AT_ONCE];
    uint4 v[AT_ONCE], w[AT_ONCE];
    int g = part * AT_ONCE, t = 0, h = 0;
    const T *from = nullptr;
    T *to = nullptr;
    bool step = false;            // the next group is the next of the same tensor: its place is a step away
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
        src[u] = nullptr;
        if (!step) {
            while (t < p.tensors - 1 && g >= p.groups_of[t]) g -= p.groups_of[t++];
            h = g * at_once + sub;
            from = (const T *)p.x[t].ptr + b * p.x[t].sb + l * p.x[t].sl + h * p.x[t].sh + c * N;
            to = (T *)p.out[t] + b * p.ob[t] + l * p.ol[t] + h * p.oh[t] + c * N;
        }
        if (sub < at_once && h < p.heads[t]) {
            src[u] = from;
            dst[u] = to;
            v[u] = *reinterpret_cast<const uint4 *>(from);
            if (!INTER) w[u] = *reinterpret_cast<const uint4 *>(from + p.pairs);
        }
        step = ++g < p.groups_of[t];
        h += at_once;
        from += at_once * p.x[t].sh;
        to += at_once * p.oh[t];
    }
    const int32_t *pos = p.positions + b * p.psb + l * p.psl;
    float2 turn[TURNS];
    ar_turns<TURNS>(p, pos, sub < at_once ? c * TURNS : p.pairs, turn);
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
        if (!src[u]) continue;
        float x[N], y[N], r[N], s[N];
        V::get(v[u], x);
        if (INTER) {
#pragma unroll
            for (int i = 0; i < TURNS; ++i) {
                const bool turned = ALL || c * TURNS + i < p.pairs;
                r[2 * i] = turned ? fmaf(x[2 * i], turn[i].x, -x[2 * i + 1] * turn[i].y) : x[2 * i];
                r[2 * i + 1] = turned ? fmaf(x[2 * i], turn[i].y, x[2 * i + 1] * turn[i].x) : x[2 * i + 1];
            }
            *reinterpret_cast<uint4 *>(dst[u]) = V::put(r);
        } else {
            V::get(w[u], y);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                r[i] = fmaf(x[i], turn[i].x, -y[i] * turn[i].y);
                s[i] = fmaf(x[i], turn[i].y, y[i] * turn[i].x);
            }
            *reinterpret_cast<uint4 *>(dst[u]) = V::put(r);
            *reinterpret_cast<uint4 *>(dst[u] + p.pairs) = V::put(s);
            // channels behind the turned ones
            for (int d = 2 * p.pairs; d < p.D - c * N; d += p.pairs)
                *reinterpret_cast<uint4 *>(dst[u] + d) = *reinterpret_cast<const uint4 *>(src[u] + d);
        }
    }
}

// Any head_dim and alignment: a thread per pair or single channel.
template <typename T, bool INTER>
__global__ void __launch_bounds__(256)
axial_rope_kernel(const __grid_constant__ AxialRope p) {
    pdl_wait();
    const int slots = p.D - p.pairs;                 // pairs, then the channels behind them
    long long heads = 0;
    for (int t = 0; t < p.tensors; ++t) heads += p.heads[t];
    const long long all = p.tokens * heads * slots;
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < all; e += (long long)gridDim.x * 256) {
        const long long row = e / slots, token = row / heads;
        const int slot = (int)(e - row * slots), b = (int)(token / p.L), l = (int)(token - (long long)b * p.L);
        int h = (int)(row - token * heads), t = 0;
        while (h >= p.heads[t]) h -= p.heads[t++];
        const T *src = (const T *)p.x[t].ptr + b * p.x[t].sb + l * p.x[t].sl + h * p.x[t].sh;
        T *dst = (T *)p.out[t] + b * p.ob[t] + l * p.ol[t] + h * p.oh[t];
        if (slot >= p.pairs) {
            dst[slot + p.pairs] = src[slot + p.pairs];
            continue;
        }
        const float2 turn = ar_turn(p, p.positions + b * p.psb + l * p.psl, slot);
        const int i = INTER ? 2 * slot : slot, j = INTER ? i + 1 : i + p.pairs;
        const float x = (float)src[i], y = (float)src[j];
        dst[i] = (T)fmaf(x, turn.x, -y * turn.y);
        dst[j] = (T)fmaf(x, turn.y, y * turn.x);
    }
}

}  // namespace wa

using namespace wa;

extern "C" int wa_axial_rope(const wa_tensor4 *x, const wa_tensor4 *out, const int32_t *heads, int tensors, int B, int L, int D,
                             const int32_t *positions, int64_t position_stride_b, int64_t position_stride_l, const int32_t *axis_pairs, int axes,
                             const float *table, int table_rows, int interleaved, int inverse, void *stream) {
    const char *what = "wa_axial_rope";
    WA_REQUIRE(x && out && heads && axis_pairs, WA_ERR_ARG, "%s: null pointer", what);
    WA_REQUIRE(tensors > 0 && tensors <= AR_TENSORS, WA_ERR_UNSUPPORTED, "%s: takes 1 to %d tensors, got %d", what, AR_TENSORS, tensors);
    WA_REQUIRE(axes > 0 && axes <= AR_AXES, WA_ERR_UNSUPPORTED, "%s: takes 1 to %d axes, got %d", what, AR_AXES, axes);
    WA_REQUIRE(B >= 0 && L >= 0 && D > 0 && table_rows > 0, WA_ERR_ARG, "%s: sizes must be positive", what);
    AxialRope p{};
    p.tensors = tensors; p.D = D; p.axes = axes; p.rows = table_rows; p.L = L; p.tokens = (long long)B * L;
    p.positions = positions; p.psb = position_stride_b; p.psl = position_stride_l;
    p.table = (const float2 *)table; p.sign = inverse ? -1.f : 1.f;
    long long pairs = 0;
    for (int a = 0; a < axes; ++a) {
        WA_REQUIRE(axis_pairs[a] >= 0, WA_ERR_ARG, "%s: an axis has %d pairs", what, axis_pairs[a]);
        pairs += axis_pairs[a];
        WA_REQUIRE(2 * pairs <= D, WA_ERR_ARG, "%s: more pairs than half the %d channels of a head", what, D);
        p.end[a] = (int)pairs;
    }
    WA_REQUIRE(pairs > 0, WA_ERR_ARG, "%s: no axis has a pair", what);
    p.pairs = (int)pairs;
    p.wide = pairs % 2 == 0 && (uintptr_t)table % 16 == 0;
    const int dtype = x[0].dtype;
    WA_REQUIRE(valid_dtype(dtype), WA_ERR_ARG, "%s: bad dtype %d", what, dtype);
    const int n = 16 / (int)dtype_size(dtype), unit = interleaved ? D : (int)pairs;      // channels of a vector; of what a head's lanes share
    bool vec = D % n == 0 && unit % n == 0 && unit / n <= 32;
    if (!interleaved) vec = vec && (D - 2 * pairs) % n == 0;
    long long all_heads = 0, groups = 0;
    for (int t = 0; t < tensors; ++t) {
        WA_REQUIRE(x[t].dtype == dtype && out[t].dtype == dtype, WA_ERR_ARG, "%s: the tensors must have one dtype", what);
        WA_REQUIRE(heads[t] >= 0, WA_ERR_ARG, "%s: sizes must be positive", what);
        WA_REQUIRE((x[t].ptr && out[t].ptr) || p.tokens * heads[t] == 0, WA_ERR_ARG, "%s: null pointer", what);
        p.x[t] = make_view(&x[t]);
        p.out[t] = out[t].ptr; p.ob[t] = out[t].stride_b; p.ol[t] = out[t].stride_l; p.oh[t] = out[t].stride_h;
        p.heads[t] = heads[t];
        all_heads += heads[t];
        if (vec) groups += p.groups_of[t] = ceil_div(heads[t], 32 / (unit / n));
        const uintptr_t places = (uintptr_t)x[t].ptr | (uintptr_t)out[t].ptr;
        const int64_t steps = x[t].stride_b | x[t].stride_l | x[t].stride_h | out[t].stride_b | out[t].stride_l | out[t].stride_h;
        vec = vec && places % 16 == 0 && steps % n == 0;
    }
    if (p.tokens == 0 || all_heads == 0) return 0;
    WA_REQUIRE(positions && table, WA_ERR_ARG, "%s: null pointer", what);
    WA_REQUIRE((uintptr_t)table % 8 == 0 && (uintptr_t)positions % 4 == 0, WA_ERR_ALIGN, "%s: the table must be 8-byte aligned", what);
    cudaError_t e;
    if (vec && B <= 65535 && groups <= 65535) {
        const int each = ar_groups(interleaved != 0);
        const bool whole = 2 * pairs == D;
        const auto kernel = dtype == WA_BF16 ? (!interleaved ? axial_rope_vec_kernel<__nv_bfloat16, false, true>
                                                : whole ? axial_rope_vec_kernel<__nv_bfloat16, true, true> : axial_rope_vec_kernel<__nv_bfloat16, true, false>)
                                             : (!interleaved ? axial_rope_vec_kernel<float, false, true>
                                                : whole ? axial_rope_vec_kernel<float, true, true> : axial_rope_vec_kernel<float, true, false>);
        e = launch_dependent(kernel, dim3(ceil_div(L, AR_WARPS), (unsigned)((groups + each - 1) / each), B), dim3(AR_WARPS * 32), 0, (cudaStream_t)stream, p);
    } else {
        const long long want = (p.tokens * all_heads * (D - pairs) + 255) / 256, most = 32ll * sm_count();
        const auto kernel = dtype == WA_BF16 ? (interleaved ? axial_rope_kernel<__nv_bfloat16, true> : axial_rope_kernel<__nv_bfloat16, false>)
                                             : (interleaved ? axial_rope_kernel<float, true> : axial_rope_kernel<float, false>);
        e = launch_dependent(kernel, dim3((unsigned)(want < most ? want : most)), dim3(256), 0, (cudaStream_t)stream, p);
    }
    if (e != cudaSuccess) return fail((int)e, "%s: %s", what, cudaGetErrorString(e));
    return check_launch(what);
}
