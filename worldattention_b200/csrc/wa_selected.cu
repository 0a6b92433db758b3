// Attention over selected key blocks with its gradient: entry points, the preparation of the lists, the form for a few query rows, and the
// gradient for every shape that the tensor-core kernels (wa_hsa_sm100.cu, wa_selected_sm100.cu) do not cover.
//
// Stands in for the autograd function of wan/modules/hsa/block_sparse_triton.py:142-382.  Its dQ kernel walks the query blocks and its dK/dV
// kernel the key blocks; so do these, so that every gradient is a sum in a fixed order in one CTA's registers and nothing is added
// atomically.  The price is that scores and dP are computed twice (seven products instead of five).
#include "wa_selected.cuh"

namespace wa {

// ---- lists ---------------------------------------------------------------------------------------
// A warp per list: ids outside the key blocks, of blocks without a key and repeated ones are dropped, the others keep their order (a router's best
// block first).  `as_listed`: repeated ids stay, those outside become the nearest block, only blocks without a key are dropped.  So a row without a
// key has an empty list, and whatever its dout holds meets no product.
// For the gradient the same ids turned around: bit i of `rows` of a key block says that query block i lists it.  Bits are set atomically, which is
// the same in any order; how often a list names the block is counted where it is met.
constexpr int SL_WARPS = 8, SL_WORDS = 1024;   // lists of a CTA; words of a bitmap up to which it has so many (32 768 key blocks)

struct SelectedLists {
    const int32_t *index, *num, *sizes;                          // sizes: keys of each key block, or null
    long long lists;
    int Nq, Nkv, stride, H, group, words, row_words, warps;      // warps: lists of a CTA
    int as_listed;
    int32_t *clean, *clean_num;
    uint32_t *rows;                                              // or null
};

__device__ __forceinline__ void selected_list(const SelectedLists &p, uint32_t *all_bits, int cta) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long list = (long long)cta * p.warps + warp;
    if (warp >= p.warps || list >= p.lists) return;
    uint32_t *bits = all_bits + (size_t)warp * p.words;
    for (int w = lane; w < p.words; w += 32) bits[w] = 0u;
    __syncwarp();
    const int n = max(0, min(p.num[list], p.stride));
    const long long bh = list / p.Nq;
    const int i = (int)(list - bh * p.Nq), h = (int)(bh % p.H), hh = h % p.group;
    const long long bhk = bh / p.H * (p.H / p.group) + h / p.group;
    int at = 0;
    for (int c = 0; c < n; c += 32) {
        int id = c + lane < n ? p.index[list * p.stride + c + lane] : -1;
        if (p.as_listed && c + lane < n) id = max(0, min(id, p.Nkv - 1));
        const bool there = (unsigned)id < (unsigned)p.Nkv && (!p.sizes || __ldg(p.sizes + id) > 0);
        const unsigned same = __match_any_sync(0xffffffffu, there ? id : -1 - lane);
        const bool take = there && (p.as_listed || (lane == __ffs(same) - 1 && !((bits[id >> 5] >> (id & 31)) & 1u)));
        __syncwarp();
        const unsigned all = __ballot_sync(0xffffffffu, take);
        if (take) {
            p.clean[list * p.stride + at + __popc(all & ((1u << lane) - 1u))] = id;
            atomicOr(&bits[id >> 5], 1u << (id & 31));
            if (p.rows) atomicOr(&p.rows[((bhk * p.Nkv + id) * p.group + hh) * p.row_words + (i >> 5)], 1u << (i & 31));
        }
        at += __popc(all);
        __syncwarp();
    }
    if (lane == 0) p.clean_num[list] = at;
}

__global__ void __launch_bounds__(SL_WARPS * 32)
selected_lists_kernel(const SelectedLists p) {
    extern __shared__ uint32_t sl_bits[];
    pdl_wait();
    selected_list(p, sl_bits, blockIdx.x);
}

// ---- work order of the gradient ------------------------------------------------------------------------
// Query blocks by the length of their lists and key blocks by the number of query blocks that list them, heaviest first: with a few items per SM
// whichever comes last otherwise works alone (see selected_ordered).  One CTA each.
__global__ void __launch_bounds__(1024)
selected_order_kernel(const int32_t *__restrict__ num, const uint32_t *__restrict__ rows, int q_items, int k_items, int words, int most_q, int most_k,
                      int32_t *__restrict__ q_order, int32_t *__restrict__ k_order) {
    __shared__ int hist[SCHED_BINS], warp_tot[32], unused[2];
    pdl_wait();
    if (blockIdx.x == 0) {
        sort_items([&](int i) { return __ldg(num + i); }, q_items, most_q, hist, warp_tot, q_order, unused, unused + 1);
    } else {
        const auto listed = [&](int i) {
            int n = 0;
            for (int w = 0; w < words; ++w) n += __popc(__ldg(rows + (long long)i * words + w));
            return n;
        };
        sort_items(listed, k_items, most_k, hist, warp_tot, k_order, unused, unused + 1);
    }
}

// ---- a few query rows ----------------------------------------------------------------------------------
// Single tokens, or up to eight rows of one query block, bf16 with head_dim 128: no tensor-core tile would be filled, and what counts is how soon the
// listed keys and values are read.  A cluster of up to eight CTAs shares a (batch, head)'s list.  Four tokens are half a warp's step: each
// token's 256 bytes are its 16 lanes' 16-byte loads, four of keys and four of values on their way at a time (eight of each take the registers of
// a third CTA per SM: 12.9 -> 18.5 us).  Scores by shuffles, a running maximum and sum per half warp; halves, warps and CTAs are joined at the end in
// a fixed order, through shared memory and the cluster's.  Every CTA cleans the list for itself (a launch less).  Float32 throughout, nothing is
// rounded but the result.
constexpr int SR_WARPS = 8, SR_STEP = 4, SR_IDS = 1024, SR_WORDS = 1024;      // tokens of a step; longest list and bitmap (32 768 key blocks)

__device__ __forceinline__ float sr_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void sr_unpack(uint4 w, float (&f)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(u[i] << 16), f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
}

template <int R>
__global__ void __launch_bounds__(SR_WARPS * 32)
selected_rows_kernel(View4 q, View4 k, View4 v, void *out, long long osb, long long osl, long long osh, float *__restrict__ lse, const int32_t *__restrict__ index,
                     const int32_t *__restrict__ num, int stride, int H, int group, int Lq, int Lkv, int block, int Nkv, float scale_log2) {
    extern __shared__ uint32_t sr_smem[];
    int32_t *ids = reinterpret_cast<int32_t *>(sr_smem);                   // [stride]
    uint32_t *bits = sr_smem + stride;                                       // [words]
    __shared__ float top_s[SR_WARPS][R], sum_s[SR_WARPS][R], acc_s[SR_WARPS][R][128];
    __shared__ float top_c[R], sum_c[R], acc_c[R][128];                      // the CTA's
    __shared__ int count;
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = lane >> 4, c = (lane & 15) * 8;
    const int h = blockIdx.y, b = blockIdx.z, hk = h / group, words = (Nkv + 31) >> 5;
    const long long list = (long long)b * H + h;
    // the query rows, scaled; rows that are none stay zero
    float qf[R][8];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        uint4 w = make_uint4(0u, 0u, 0u, 0u);
        if (r < Lq) w = *reinterpret_cast<const uint4 *>((const __nv_bfloat16 *)q.ptr + b * q.sb + r * q.sl + h * q.sh + c);
        sr_unpack(w, qf[r]);
#pragma unroll
        for (int e = 0; e < 8; ++e) qf[r][e] *= scale_log2;
    }
    for (int w = threadIdx.x; w < words; w += SR_WARPS * 32) bits[w] = 0u;
    __syncthreads();
    if (warp == 0) {
        const int n = max(0, min(num[list], stride));
        int at = 0;
        for (int i = 0; i < n; i += 32) {
            const int id = i + lane < n ? index[list * stride + i + lane] : -1;
            const bool there = (unsigned)id < (unsigned)Nkv;
            const unsigned same = __match_any_sync(0xffffffffu, there ? id : -1 - lane);
            const bool take = there && lane == __ffs(same) - 1 && !((bits[id >> 5] >> (id & 31)) & 1u);
            __syncwarp();
            const unsigned all = __ballot_sync(0xffffffffu, take);
            if (take) {
                ids[at + __popc(all & ((1u << lane) - 1u))] = id;
                atomicOr(&bits[id >> 5], 1u << (id & 31));
            }
            at += __popc(all);
            __syncwarp();
        }
        if (lane == 0) count = at;
    }
    __syncthreads();
    float top[R], sum[R], acc[R][8];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        top[r] = -INFINITY;
        sum[r] = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[r][e] = 0.f;
    }
    const __nv_bfloat16 *kp = (const __nv_bfloat16 *)k.ptr + b * k.sb + hk * k.sh + c, *vp = (const __nv_bfloat16 *)v.ptr + b * v.sb + hk * v.sh + c;
    const int per_block = block / SR_STEP, steps = count * per_block;        // (block is 64 or 128)
    const int step0 = (blockIdx.x * SR_WARPS + warp) * 2, all_steps = gridDim.x * SR_WARPS * 2;
    for (int s0 = step0; s0 < steps; s0 += all_steps) {                       // both halves of a warp stay together
        const int s = s0 + half;
        const int e0 = s < steps ? s / per_block : 0, token0 = s < steps ? ids[e0] * block + (s - e0 * per_block) * SR_STEP : Lkv;
        uint4 kw[SR_STEP], vw[SR_STEP];
#pragma unroll
        for (int t = 0; t < SR_STEP; ++t) {
            kw[t] = vw[t] = make_uint4(0u, 0u, 0u, 0u);
            if (token0 + t < Lkv) {
                kw[t] = __ldg(reinterpret_cast<const uint4 *>(kp + (token0 + t) * k.sl));
                vw[t] = __ldg(reinterpret_cast<const uint4 *>(vp + (token0 + t) * v.sl));
            }
        }
        float z[R][SR_STEP];
#pragma unroll
        for (int t = 0; t < SR_STEP; ++t) {
            float kf[8];
            sr_unpack(kw[t], kf);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float d = qf[r][0] * kf[0];
#pragma unroll
                for (int e = 1; e < 8; ++e) d = fmaf(qf[r][e], kf[e], d);
                z[r][t] = d;
            }
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1)
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int t = 0; t < SR_STEP; ++t) z[r][t] += __shfl_xor_sync(0xffffffffu, z[r][t], o);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float high = top[r];
#pragma unroll
            for (int t = 0; t < SR_STEP; ++t) {
                if (token0 + t >= Lkv) z[r][t] = -INFINITY;
                high = fmaxf(high, z[r][t]);
            }
            const float at = high == -INFINITY ? 0.f : high, back = sr_exp2(top[r] - at);      // (nothing seen yet: 2^-inf = 0)
            top[r] = high;
            sum[r] *= back;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[r][e] *= back;
#pragma unroll
            for (int t = 0; t < SR_STEP; ++t) {
                z[r][t] = sr_exp2(z[r][t] - at);
                sum[r] += z[r][t];
            }
        }
#pragma unroll
        for (int t = 0; t < SR_STEP; ++t) {
            float vf[8];
            sr_unpack(vw[t], vf);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[r][e] = fmaf(z[r][t], vf[e], acc[r][e]);
        }
    }
    // halves of a warp
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float other = __shfl_xor_sync(0xffffffffu, top[r], 16), high = fmaxf(top[r], other), at = high == -INFINITY ? 0.f : high;
        const float mine = sr_exp2(top[r] - at);
        sum[r] *= mine;
        sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 16);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            acc[r][e] *= mine;
            acc[r][e] += __shfl_xor_sync(0xffffffffu, acc[r][e], 16);
            if (half == 0) acc_s[warp][r][c + e] = acc[r][e];
        }
        if (lane == 0) top_s[warp][r] = high, sum_s[warp][r] = sum[r];
    }
    __syncthreads();
    // warps of the CTA
    for (int i = threadIdx.x; i < R * 128; i += SR_WARPS * 32) {
        const int r = i >> 7, d = i & 127;
        float high = -INFINITY, total = 0.f, x = 0.f;
#pragma unroll
        for (int w = 0; w < SR_WARPS; ++w) high = fmaxf(high, top_s[w][r]);
        const float at = high == -INFINITY ? 0.f : high;
#pragma unroll
        for (int w = 0; w < SR_WARPS; ++w) {
            const float f = sr_exp2(top_s[w][r] - at);
            total = fmaf(sum_s[w][r], f, total);
            x = fmaf(acc_s[w][r][d], f, x);
        }
        acc_c[r][d] = x;
        if (d == 0) top_c[r] = high, sum_c[r] = total;
    }
    // CTAs of the cluster: CTA j joins rows j, j + CTAs, ...
    const int ctas = gridDim.x;
    if (ctas > 1) {
        asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    } else {
        __syncthreads();
    }
    const auto far = [](const float *p, int cta) {
        float x;
        uint32_t at;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(cta));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(at) : "memory");
        return x;
    };
    for (int r = blockIdx.x; r < Lq; r += ctas) {
        const int d = threadIdx.x;
        if (d >= 128) continue;
        float tops[8], high = -INFINITY, total = 0.f, x = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) tops[j] = j < ctas ? far(&top_c[r], j) : -INFINITY, high = fmaxf(high, tops[j]);
        const float at = high == -INFINITY ? 0.f : high;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < ctas) {
                const float f = sr_exp2(tops[j] - at);
                total = fmaf(far(&sum_c[r], j), f, total);
                x = fmaf(far(&acc_c[r][d], j), f, x);
            }
        // (no key: zero and -inf; a sum that is not a number stays one)
        ((__nv_bfloat16 *)out)[b * osb + r * osl + h * osh + d] = __float2bfloat16_rn(total == 0.f ? 0.f : x / total);
        if (lse && d == 0) lse[list * Lq + r] = total == 0.f ? -INFINITY : (high + log2f(total)) * 0.6931471805599453f;
    }
    if (ctas > 1) {      // the others may still be reading
        asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    }
}

static bool selected_few_rows(const wa_selected_params *p) {
    const auto pieces = [](const wa_tensor4 &t) { return (uintptr_t)t.ptr % 16 == 0 && t.stride_b % 8 == 0 && t.stride_l % 8 == 0 && t.stride_h % 8 == 0; };
    return p->q.dtype == WA_BF16 && p->D == 128 && p->Lq <= 8 && (p->block_size == 64 || p->block_size == 128) && !p->block_sizes && p->index_stride <= SR_IDS &&
           ceil_div(p->Lkv, p->block_size) <= 32 * SR_WORDS && pieces(p->q) && pieces(p->k) && pieces(p->v);
}

static int launch_few_rows(const wa_selected_params *p, cudaStream_t stream) {
    const char *what = "wa_selected_forward";
    const int Nkv = ceil_div(p->Lkv, p->block_size);
    // as many CTAs for a list as it has work for, up to about four for every SM (4 x 12 lists of 32 blocks: 8 CTAs each 12.9 us, 4 14.2)
    int ctas = 8;
    const long long lists = (long long)p->B * p->H, steps = (long long)p->index_stride * p->block_size / SR_STEP;
    while (ctas > 1 && (lists * ctas > 4ll * sm_count() || (long long)ctas * SR_WARPS * 2 > steps)) ctas >>= 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas, p->H, p->B);
    cfg.blockDim = dim3(SR_WARPS * 32);
    cfg.dynamicSmemBytes = ((size_t)p->index_stride + ceil_div(Nkv, 32)) * 4;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    const float scale = (float)(1.4426950408889634 / sqrt(128.0));
    const auto kernel = p->Lq == 1 ? selected_rows_kernel<1> : p->Lq == 2 ? selected_rows_kernel<2> : p->Lq <= 4 ? selected_rows_kernel<4> : selected_rows_kernel<8>;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, make_view(&p->q), make_view(&p->k), make_view(&p->v), p->out.ptr, (long long)p->out.stride_b,
                                             (long long)p->out.stride_l, (long long)p->out.stride_h, p->lse, p->index, p->num, p->index_stride, p->H, p->H / p->Hkv, p->Lq,
                                             p->Lkv, p->block_size, Nkv, scale);
    if (e != cudaSuccess) return fail((int)e, "%s: %s", what, cudaGetErrorString(e));
    return check_launch(what);
}

// The bits that the lists set, and the counters of the tensor-core kernels behind them.  (As a memset between two kernels: 4.5 us instead of 1.5.)
__global__ void __launch_bounds__(256)
selected_zeros_kernel(uint4 *to, size_t pieces) {
    pdl_wait();
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < pieces; i += (size_t)gridDim.x * 256) to[i] = make_uint4(0u, 0u, 0u, 0u);
}

static int launch_zeros(char *to, size_t bytes, cudaStream_t stream, const char *what) {       // both multiples of 16
    const size_t pieces = bytes / 16, want = (pieces + 255) / 256, most = 8 * (size_t)sm_count();
    const cudaError_t e = launch_dependent(selected_zeros_kernel, dim3((unsigned)(want < most ? want : most)), dim3(256), 0, stream, (uint4 *)to, pieces);
    if (e != cudaSuccess) return fail((int)e, "%s: %s", what, cudaGetErrorString(e));
    return check_launch(what);
}

// ---- row statistics of the gradient -----------------------------------------------------------------
// See selected_stat.  Reads dout and out once: `LANES` lanes take a row, 16 bytes each (LANES = 0: a warp, one channel at a time, any layout), and
// four rows are on their way at a time.  The first CTAs of the launch clean the lists, which nothing here needs.
template <typename T, int LANES>
__global__ void __launch_bounds__(256)
selected_prepare_kernel(const SelectedLists lists, unsigned list_ctas, View4 out, View4 dout, const float *__restrict__ lse, int H, int Lq, int D, int padded, unsigned all,
                        float *__restrict__ stats) {
    extern __shared__ uint32_t sl_bits[];
    pdl_wait();
    if (blockIdx.x < list_ctas) {
        if (blockIdx.y == 0) selected_list(lists, sl_bits, blockIdx.x);
        return;
    }
    constexpr int WIDE = LANES ? LANES : 32, AT_ONCE = LANES ? 4 : 1, N = 16 / sizeof(T), EACH = 256 / WIDE;
    const int sub = threadIdx.x / WIDE, lane = threadIdx.x % WIDE, b = blockIdx.y;
    unsigned row[AT_ONCE];                        // (token, h) of the sample, heads innermost as in memory
    int h[AT_ONCE], l[AT_ONCE];
    float sum[AT_ONCE], natural[AT_ONCE];
    uint4 x[AT_ONCE], y[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
        row[u] = ((blockIdx.x - list_ctas) * AT_ONCE + u) * EACH + sub;
        l[u] = (int)(row[u] / (unsigned)H);
        h[u] = (int)(row[u] - (unsigned)l[u] * (unsigned)H);
        sum[u] = 0.f;
        if (row[u] >= all || l[u] >= Lq) continue;
        natural[u] = __ldg(lse + ((long long)b * H + h[u]) * Lq + l[u]);
        const T *o = (const T *)out.ptr + b * out.sb + (long long)l[u] * out.sl + (long long)h[u] * out.sh;
        const T *g = (const T *)dout.ptr + b * dout.sb + (long long)l[u] * dout.sl + (long long)h[u] * dout.sh;
        if (LANES) {
            x[u] = __ldg(reinterpret_cast<const uint4 *>(o) + lane);
            y[u] = __ldg(reinterpret_cast<const uint4 *>(g) + lane);
        } else {
            for (int d = lane; d < D; d += 32) sum[u] = fmaf((float)o[d], (float)g[d], sum[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
        const bool there = row[u] < all && l[u] < Lq;
        if (LANES && there) {
            const T *a = reinterpret_cast<const T *>(&x[u]), *c = reinterpret_cast<const T *>(&y[u]);
#pragma unroll
            for (int e = 0; e < N; ++e) sum[u] = fmaf((float)a[e], (float)c[e], sum[u]);
        }
#pragma unroll
        for (int o = WIDE / 2; o > 0; o >>= 1) sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], o);
        if (lane == 0 && row[u] < all) {
            // a row behind the last one, or one that nothing is listed for: no key sees it
            const bool seen = there && natural[u] != -INFINITY;
            float *to = stats + ((long long)b * H + h[u]) * padded * 2 + selected_stat(l[u]);
            to[0] = seen ? -1.4426950408889634f * natural[u] : -INFINITY;
            to[64] = seen ? -sum[u] : 0.f;
        }
    }
}

template <typename T>
static int launch_prepare(const wa_selected_params *p, const SelectedLists &lists, int padded, float *stats, cudaStream_t stream) {
    const char *what = "wa_selected_backward";
    const auto pieces = [](const wa_tensor4 &t) {       // rows of whole 16-byte pieces
        constexpr int n = 16 / sizeof(T);
        return (uintptr_t)t.ptr % 16 == 0 && t.stride_b % n == 0 && t.stride_l % n == 0 && t.stride_h % n == 0;
    };
    const int bytes = p->D * (int)sizeof(T), lanes = pieces(p->out) && pieces(p->dout) && (bytes == 512 || bytes == 256 || bytes == 128) ? bytes / 16 : 0;
    const long long all = (long long)p->H * padded, each = lanes ? 4 * (256 / lanes) : 8, list_ctas = (lists.lists + lists.warps - 1) / lists.warps;
    WA_REQUIRE(all + 1024 < (1ll << 32) && list_ctas + (all + each - 1) / each < (1ll << 31), WA_ERR_UNSUPPORTED, "%s: too many tokens", what);
    const auto kernel = lanes == 32 ? selected_prepare_kernel<T, 32> : lanes == 16 ? selected_prepare_kernel<T, 16> : lanes == 8 ? selected_prepare_kernel<T, 8> : selected_prepare_kernel<T, 0>;
    const size_t smem = (size_t)lists.warps * lists.words * sizeof(uint32_t);
    static PerDeviceOnce attr_set;
    if (smem > 48 * 1024 && !attr_set.done()) {
        for (auto k : {selected_prepare_kernel<T, 32>, selected_prepare_kernel<T, 16>, selected_prepare_kernel<T, 8>, selected_prepare_kernel<T, 0>}) {
            const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, 192 * 1024);
            if (e != cudaSuccess) return fail((int)e, "%s: %s", what, cudaGetErrorString(e));
        }
        attr_set.mark();
    }
    const cudaError_t e = launch_dependent(kernel, dim3((unsigned)(list_ctas + (all + each - 1) / each), p->B), dim3(256), smem, stream, lists, (unsigned)list_ctas,
                                           make_view(&p->out), make_view(&p->dout), p->lse, p->H, p->Lq, p->D, padded, (unsigned)all, stats);
    if (e != cudaSuccess) return fail((int)e, "%s: %s", what, cudaGetErrorString(e));
    return check_launch(what);
}

// ---- any shape -----------------------------------------------------------------------------------------
// Forward and gradient with multiply-adds, for what the tensor-core kernels do not take.  One CTA owns TF rows of one side -- forward and dQ: queries,
// dK/dV: keys -- and meets the rows of the other side TG at a time.  A warp has TF / 8 of the owned rows to itself: its lanes take TG / 32 met
// rows each for the scores, P and dS go through shared memory of the warp's own, and for the sums a lane has CH channels (the width is 32 CH:
// 64, 128 or 256).  So an owned row is one address for all lanes, a met row one for each, both 16 bytes: with 64 and 64 rows 16 wavefronts of shared
// memory for 64 multiply-adds of a warp (scores), 24 for 128 (sums), below what the multiply-adds take.  (16 x 16 threads with 2 x 2 scores each were
// bound by shared memory: three frames of 390 tokens, 12 heads, 3 of 19 blocks of 64 a row: dK/dV 187 us and dQ 143, now 161 and 119, heaviest first
// 141 and 85.)  Where 64 owned rows leave SMs without a CTA there are 32 or 16 to a CTA, see selected_own.
// The next rows to meet are on their way while some are at work: asynchronous copies of aligned float32 rows, plain loads of anything else.
struct SelectedAny {
    View4 q, k, v, dout;
    void *out, *dq, *dk, *dv;
    float *lse;
    int dtype;
    long long ob, ol, oh, dqb, dql, dqh, dkb, dkl, dkh, dvb, dvl, dvh;
    int H, group, Lq, Lkv, D, block, stride, Nq, Nkv, row_words, padded, tiles;
    int async;                        // rows of whole 16-byte pieces of float32
    int as_listed;                    // a query block's list may name a key block more than once
    const int32_t *index, *num, *block_sizes;
    const int32_t *q_order, *k_order; // or null: as they come
    const uint32_t *rows;
    const float *stats;
    float scale;
};
enum { SG_FORWARD, SG_QUERIES, SG_KEYS };

// channels of a lane: CH neighbouring ones, or four of each half of 256
template <int CH>
__device__ __forceinline__ void sg_channels(const float *row, int lane, float (&y)[CH]) {
    if constexpr (CH == 2) {
        const float2 v = *reinterpret_cast<const float2 *>(row + 2 * lane);
        y[0] = v.x, y[1] = v.y;
    } else {
#pragma unroll
        for (int m = 0; m < CH / 4; ++m) {
            const float4 v = *reinterpret_cast<const float4 *>(row + 128 * m + 4 * lane);
            y[4 * m] = v.x, y[4 * m + 1] = v.y, y[4 * m + 2] = v.z, y[4 * m + 3] = v.w;
        }
    }
}
template <int CH>
__device__ __forceinline__ int sg_channel(int lane, int u) { return CH == 2 ? 2 * lane + u : 128 * (u >> 2) + 4 * lane + (u & 3); }

template <int TF, int TG, int CH>
constexpr size_t sg_smem(int what) {
    return (size_t)(((what == SG_FORWARD ? 1 : 2) * TF + 4 * TG) * (32 * CH + 4) + TF * (TG + 4)) * 4 + 2 * (size_t)(TF > TG ? TF : TG) * 8;
}

template <int TF, int TG, int CH, int WHAT>
__global__ void __launch_bounds__(256)
selected_any_kernel(const SelectedAny p) {
    constexpr bool KEYS = WHAT == SG_KEYS, FORWARD = WHAT == SG_FORWARD;
    constexpr int W = 32 * CH, LD = W + 4, R = TF / 8, C = TG / 32, LP = TG + 4;      // R: owned rows of a warp, C: met rows of a lane
    constexpr int ST = TF > TG ? TF : TG;
    // Two multiply-adds an instruction where a warp has eight rows: issue slots count beside shared memory there (12 heads of 1170 tokens, dK/dV 127 -> 118 us;
    // eight of 1500, head_dim 64, dQ 158 -> 151, its forward 83 -> 79).  With fewer rows the chains get too long (64 queries, dQ 81 -> 85), and so they do
    // in the forward of head_dim 128 (62 -> 65).
    constexpr bool TWO = TF == 64 && (WHAT != SG_FORWARD || CH == 2);
    extern __shared__ __align__(16) float sg_smem_[];
    float *f1 = sg_smem_, *f2 = f1 + TF * LD, *met = FORWARD ? f2 : f2 + TF * LD;     // owned: q (and dout) or k, v; met: [two buffers][the other two]
    float *factors = met + 4 * TG * LD;                                                // P, then dS
    float2 *st = reinterpret_cast<float2 *>(factors + TF * LP);                        // [two buffers] statistics of the query rows
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (WHAT != SG_QUERIES) pdl_wait();         // (dQ waits at its end: see wa_selected_backward)
    if (KEYS) pdl_release_dependents();
    const int blocks = KEYS ? p.Nkv : p.Nq, heads = KEYS ? p.H / p.group : p.H;
    const int32_t *order = KEYS ? p.k_order : p.q_order;
    const int item = order ? order[blockIdx.x / p.tiles] : blockIdx.x / p.tiles, own_head = item / blocks;
    const int blk = item - own_head * blocks, first = blk * p.block + (blockIdx.x % p.tiles) * TF, b = own_head / heads, h = own_head - b * heads;
    const int hk = KEYS ? h : h / p.group;
    const auto keys_of = [&](int id) {       // real tokens of a key block
        const int n = min(p.block, p.Lkv - id * p.block);
        return p.block_sizes ? max(0, min(n, p.block_sizes[id])) : n;
    };
    const int own_end = min(min(first + TF, (blk + 1) * p.block), KEYS ? p.Lkv : p.Lq);       // rows to write
    const int own_real = KEYS ? min(own_end, blk * p.block + keys_of(blk)) : own_end;          // rows that count
    if (first >= own_end) {
        if (WHAT == SG_QUERIES) pdl_wait();
        return;
    }

    const auto bring = [&](float *to, const View4 &x, int head, int from, int end, int rows) {
        const long long base = b * x.sb + (long long)head * x.sh;
        if (p.async) {
            for (int e = threadIdx.x; e < rows * (W / 4); e += 256) {
                const int r = e / (W / 4), d = e % (W / 4) * 4;
                const bool there = from + r < end && d < p.D;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to + r * LD + d)),
                             "l"((const float *)x.ptr + (there ? base + (long long)(from + r) * x.sl + d : 0)), "r"(there ? 16 : 0) : "memory");
            }
        } else {
#pragma unroll 4
            for (int e = threadIdx.x; e < rows * W; e += 256) {
                const int r = e / W, d = e % W;
                to[r * LD + d] = from + r < end && d < p.D ? load_elem(x.ptr, x.dtype, base + (long long)(from + r) * x.sl + d) : 0.f;
            }
        }
    };
    const auto bring_stats = [&](float2 *to, int head, int from, int end, int rows) {
        const float *stats = p.stats + ((long long)b * p.H + head) * p.padded * 2;
        for (int r = threadIdx.x; r < rows; r += 256)
            to[r] = from + r < end ? make_float2(stats[selected_stat(from + r)], stats[selected_stat(from + r) + 64]) : make_float2(-INFINITY, 0.f);
    };
    bring(f1, KEYS ? p.k : p.q, h, first, own_real, TF);
    if (!FORWARD) bring(f2, KEYS ? p.v : p.dout, h, first, own_real, TF);
    if (WHAT == SG_QUERIES) bring_stats(st, h, first, own_real, TF);

    // the rows to meet, TG at a time: those of the listed blocks in the order of the list
    struct Rows { int h, from, end; };
    int at = -1, left_from = 0, left_end = 0, head = 0, times = 1;        // times: keys, how often the list still names this block
    uint32_t word = 0;
    const long long list = KEYS ? (long long)item * p.group * p.row_words : (long long)item;
    const int n = KEYS ? p.group * p.row_words : p.num[list];
    const auto next = [&](Rows &to) {
        while (left_from >= left_end) {
            if (KEYS) {
                if (times > 1) {
                    --times;
                    left_from = (left_end - 1) / p.block * p.block;
                    continue;
                }
                while (word == 0u) {
                    if (++at >= n) return false;
                    word = p.rows[list + at];
                }
                const int i = (at % p.row_words) * 32 + __ffs(word) - 1;
                word &= word - 1;
                head = hk * p.group + at / p.row_words;
                left_from = i * p.block;
                left_end = min(left_from + p.block, p.Lq);
                if (p.as_listed) {
                    const long long row = ((long long)b * p.H + head) * p.Nq + i;
                    unsigned named = 0;
                    for (int e = lane; e < p.num[row]; e += 32) named += p.index[row * p.stride + e] == blk;
                    times = (int)__reduce_add_sync(0xffffffffu, named);
                }
            } else {
                if (++at >= n) return false;
                const int id = p.index[list * p.stride + at];
                head = h;
                left_from = id * p.block;
                left_end = left_from + keys_of(id);
            }
        }
        to = Rows{head, left_from, min(left_from + TG, left_end)};
        left_from += TG;
        return true;
    };
    const auto bring_met = [&](int buf, const Rows &r) {
        bring(met + 2 * buf * TG * LD, KEYS ? p.q : p.k, KEYS ? r.h : hk, r.from, r.end, TG);
        bring(met + (2 * buf + 1) * TG * LD, KEYS ? p.dout : p.v, KEYS ? r.h : hk, r.from, r.end, TG);
        if (KEYS) bring_stats(st + buf * ST, r.h, r.from, r.end, TG);
    };

    float sum1[R][CH], sum2[R][CH];         // of the owned rows: dV (KEYS); dK, dQ or the result
    float top[R], total[R];                 // forward: running maximum of a row, and this lane's part of the sum
#pragma unroll
    for (int i = 0; i < R; ++i) {
        top[i] = -INFINITY;
        total[i] = 0.f;
#pragma unroll
        for (int u = 0; u < CH; ++u) sum1[i][u] = sum2[i][u] = 0.f;
    }
    const float to_log2 = p.scale * 1.4426950408889634f;
    const int depth = (p.D + 3) & ~3;

    Rows now, then;
    bool more = next(now);
    if (more) bring_met(0, now);
    asm volatile("cp.async.commit_group;" ::: "memory");
    for (int buf = 0; more; buf ^= 1, now = then) {
        more = next(then);
        if (more) bring_met(buf ^ 1, then);
        asm volatile("cp.async.commit_group;" ::: "memory");
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncthreads();
        const float *g1 = met + 2 * buf * TG * LD, *g2 = g1 + TG * LD;
        float s[R][C], dp[R][C];
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < C; ++j) s[i][j] = dp[i][j] = 0.f;
        const auto dots = [&](float (&acc)[R][C], const float *f, const float *g) {
            if constexpr (TWO) {               // of even and of odd channels
                float2 two[R][C];
#pragma unroll
                for (int i = 0; i < R; ++i)
#pragma unroll
                    for (int j = 0; j < C; ++j) two[i][j] = make_float2(0.f, 0.f);
#pragma unroll 2
                for (int d = 0; d < depth; d += 4) {
                    float4 y[C];
#pragma unroll
                    for (int j = 0; j < C; ++j) y[j] = *reinterpret_cast<const float4 *>(g + (lane + 32 * j) * LD + d);
#pragma unroll
                    for (int i = 0; i < R; ++i) {
                        const float4 x = *reinterpret_cast<const float4 *>(f + (warp * R + i) * LD + d);
#pragma unroll
                        for (int j = 0; j < C; ++j) {
                            two[i][j] = __ffma2_rn(make_float2(x.x, x.y), make_float2(y[j].x, y[j].y), two[i][j]);
                            two[i][j] = __ffma2_rn(make_float2(x.z, x.w), make_float2(y[j].z, y[j].w), two[i][j]);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < R; ++i)
#pragma unroll
                    for (int j = 0; j < C; ++j) acc[i][j] = two[i][j].x + two[i][j].y;
                return;
            }
#pragma unroll 2
            for (int d = 0; d < depth; d += 4) {
                float4 y[C];
#pragma unroll
                for (int j = 0; j < C; ++j) y[j] = *reinterpret_cast<const float4 *>(g + (lane + 32 * j) * LD + d);
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const float4 x = *reinterpret_cast<const float4 *>(f + (warp * R + i) * LD + d);
#pragma unroll
                    for (int j = 0; j < C; ++j) {
                        acc[i][j] = fmaf(x.x, y[j].x, acc[i][j]);
                        acc[i][j] = fmaf(x.y, y[j].y, acc[i][j]);
                        acc[i][j] = fmaf(x.z, y[j].z, acc[i][j]);
                        acc[i][j] = fmaf(x.w, y[j].w, acc[i][j]);
                    }
                }
            }
        };
        dots(s, f1, g1);
        if (!FORWARD) dots(dp, f2, g2);
        float *mine = factors + warp * R * LP;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (FORWARD) {
                float high = top[i];
#pragma unroll
                for (int j = 0; j < C; ++j) {
                    s[i][j] = now.from + lane + 32 * j < now.end ? s[i][j] * to_log2 : -INFINITY;
                    high = fmaxf(high, s[i][j]);
                }
                high = warp_max(high);
                const float from = high == -INFINITY ? 0.f : high, back = exp2f(top[i] - from);      // (nothing seen yet: 2^-inf = 0)
                top[i] = high;
                total[i] *= back;
#pragma unroll
                for (int u = 0; u < CH; ++u) sum2[i][u] *= back;
#pragma unroll
                for (int j = 0; j < C; ++j) {
                    s[i][j] = exp2f(s[i][j] - from);
                    total[i] += s[i][j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < C; ++j) {
                    const int f = warp * R + i, g = lane + 32 * j;
                    const float2 row = st[KEYS ? buf * ST + g : f];
                    const bool there = first + f < own_real && now.from + g < now.end;
                    s[i][j] = there ? exp2f(fmaf(s[i][j], to_log2, row.x)) : 0.f;
                    dp[i][j] = there ? s[i][j] * (dp[i][j] + row.y) * p.scale : 0.f;
                }
            }
        }
        const auto add = [&](float (&acc)[R][CH], const float (&factor)[R][C], const float *x) {
            __syncwarp();
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int j = 0; j < C; ++j) mine[i * LP + lane + 32 * j] = factor[i][j];
            __syncwarp();
#pragma unroll 2
            for (int g = 0; g < TG; g += 4) {
                float y[4][CH];
#pragma unroll
                for (int u = 0; u < 4; ++u) sg_channels<CH>(x + (g + u) * LD, lane, y[u]);
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const float4 a = *reinterpret_cast<const float4 *>(mine + i * LP + g);
                    if constexpr (TWO) {
#pragma unroll
                        for (int m = 0; m < CH; m += 2) {
                            float2 t = make_float2(acc[i][m], acc[i][m + 1]);
                            t = __ffma2_rn(make_float2(a.x, a.x), make_float2(y[0][m], y[0][m + 1]), t);
                            t = __ffma2_rn(make_float2(a.y, a.y), make_float2(y[1][m], y[1][m + 1]), t);
                            t = __ffma2_rn(make_float2(a.z, a.z), make_float2(y[2][m], y[2][m + 1]), t);
                            t = __ffma2_rn(make_float2(a.w, a.w), make_float2(y[3][m], y[3][m + 1]), t);
                            acc[i][m] = t.x;
                            acc[i][m + 1] = t.y;
                        }
                    } else {
#pragma unroll
                        for (int m = 0; m < CH; ++m) {
                            acc[i][m] = fmaf(a.x, y[0][m], acc[i][m]);
                            acc[i][m] = fmaf(a.y, y[1][m], acc[i][m]);
                            acc[i][m] = fmaf(a.z, y[2][m], acc[i][m]);
                            acc[i][m] = fmaf(a.w, y[3][m], acc[i][m]);
                        }
                    }
                }
            }
        };
        if (FORWARD) {
            add(sum2, s, g2);
        } else {
            if (KEYS) add(sum1, s, g2);
            add(sum2, dp, g1);
        }
        __syncthreads();
    }
    const auto write = [&](const float (&acc)[R][CH], void *to, long long sb, long long sl, long long sh) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int r = first + warp * R + i;
            if (r >= own_end) continue;
#pragma unroll
            for (int u = 0; u < CH; ++u) {
                const int d = sg_channel<CH>(lane, u);
                if (d < p.D) store_elem(to, p.dtype, b * sb + r * sl + h * sh + d, r < own_real ? acc[i][u] : 0.f);      // (tokens that are no keys: a met row's NaN times zero)
            }
        }
    };
    if (FORWARD) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const float all = warp_sum(total[i]);
            const int r = first + warp * R + i;
#pragma unroll
            for (int u = 0; u < CH; ++u) sum2[i][u] = all == 0.f ? 0.f : sum2[i][u] / all;
            if (p.lse && lane == 0 && r < own_end) p.lse[((long long)b * p.H + h) * p.Lq + r] = all == 0.f ? -INFINITY : (top[i] + log2f(all)) * 0.6931471805599453f;
        }
        write(sum2, p.out, p.ob, p.ol, p.oh);
    } else if (KEYS) {
        write(sum1, p.dv, p.dvb, p.dvl, p.dvh);
        write(sum2, p.dk, p.dkb, p.dkl, p.dkh);
    } else {
        write(sum2, p.dq, p.dqb, p.dql, p.dqh);
        pdl_wait();
    }
}

template <int TF, int TG, int CH, int WHAT>
static int launch_any(SelectedAny p, long long items, cudaStream_t stream, const char *what) {
    constexpr size_t smem = sg_smem<TF, TG, CH>(WHAT);
    static_assert(smem <= 227 * 1024, "shared memory budget exceeded");
    static PerDeviceOnce attr_set;
    if (!attr_set.done()) {
        const cudaError_t e = cudaFuncSetAttribute(selected_any_kernel<TF, TG, CH, WHAT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return fail((int)e, "%s: %s", what, cudaGetErrorString(e));
        attr_set.mark();
    }
    p.tiles = ceil_div(p.block, TF);
    const long long ctas = items * p.tiles;
    WA_REQUIRE(ctas < (1ll << 31), WA_ERR_UNSUPPORTED, "%s: grid too large", what);
    const cudaError_t e = launch_dependent(selected_any_kernel<TF, TG, CH, WHAT>, dim3((unsigned)ctas), dim3(256), smem, stream, p);
    if (e != cudaSuccess) return fail((int)e, "%s: %s", what, cudaGetErrorString(e));
    return check_launch(what);
}

// Owned rows of a CTA: 64, 32 or 16, whichever is done first, of about equal ones the larger (it reads the met rows less often; 1170 tokens of 12
// heads, up to six blocks listed: forward, dQ and dK/dV 61, 85 and 125 us with 64, 71, 95 and 118 with 32).  A CTA of 32 rows takes 0.65 of the time of one of
// 64, one of 16 0.52 (its warps read a met row for two owned ones instead of eight), and as many rounds as its SMs take; head_dim 64 leaves room for two on
// an SM.  head_dim 128, 12 heads, 10 blocks of 64 listed, forward and dQ with 64 rows -> as chosen: 64 queries 95 and 135 us -> 51 and 68 (16 rows); 700
// 97 and 137 (64 rows; with 32 125 and 176).
static int selected_own(long long rows, int block, int limit, int resident) {
    const long long room = (long long)sm_count() * resident;
    const auto cost = [&](int own) { return ((rows + own - 1) / own + room - 1) / room * (own == 64 ? 20 : own == 32 ? 13 : 11); };
    int best = 16;
    for (int own = 32; own <= limit; own <<= 1)
        if (own < 2 * block && cost(own) * 9 <= cost(best) * 10) best = own;
    return best;
}

template <int WHAT>
static int run_any(const SelectedAny &p, int B, cudaStream_t stream, const char *what) {
    const int heads = WHAT == SG_KEYS ? p.H / p.group : p.H, blocks = WHAT == SG_KEYS ? p.Nkv : p.Nq;
    const long long items = (long long)B * heads * blocks;
    const int own = selected_own((long long)B * heads * (WHAT == SG_KEYS ? p.Lkv : p.Lq), p.block, p.D <= 128 ? 64 : 32, p.D <= 64 ? 2 : 1);
    if (p.D <= 64) return own == 64 ? launch_any<64, 64, 2, WHAT>(p, items, stream, what) : own == 32 ? launch_any<32, 64, 2, WHAT>(p, items, stream, what) : launch_any<16, 64, 2, WHAT>(p, items, stream, what);
    if (p.D <= 128) return own == 64 ? launch_any<64, 64, 4, WHAT>(p, items, stream, what) : own == 32 ? launch_any<32, 64, 4, WHAT>(p, items, stream, what) : launch_any<16, 64, 4, WHAT>(p, items, stream, what);
    return own == 32 ? launch_any<32, 32, 8, WHAT>(p, items, stream, what) : launch_any<16, 32, 8, WHAT>(p, items, stream, what);
}

// ---- host ----------------------------------------------------------------------------------------
// Heaviest first where there are more items than SMs and their tensors about fit L2 side by side: the order over all heads mixes the heads, which larger
// calls pay for with what the CTAs of one head would find in L2.  Both gradients with counts between zero and 32 blocks of 64 (16 of 128), 12 heads, bf16,
// as they come -> ordered, its launch included: 1200 tokens 51.5 -> 46.2 us, 4680 170 -> 153 (133 -> 110), 9360 (115 MB) 301 -> 293 (224 -> 195), 18 720
// 549 -> 584 (387 -> 374).  Float32: three frames of 390 tokens 282 -> 230, its forward 103 -> 77; 2900 tokens 1240 -> 971, 450 -> 354.
static bool selected_ordered(const wa_selected_params *p, const SelectedPlan &w) {
    const long long bytes = 2ll * dtype_size(p->q.dtype) * p->B * p->D * ((long long)p->H * p->Lq + (long long)p->Hkv * p->Lkv);
    return (long long)p->B * p->H * w.Nq > sm_count() && (long long)p->B * p->H * w.Nq <= (1 << 20) && (long long)p->B * p->Hkv * w.Nkv <= (1 << 20) && bytes <= 128ll << 20;
}

static SelectedPlan selected_plan(const wa_selected_params *p, bool backward) {
    SelectedPlan w{};
    w.Nq = ceil_div(p->Lq, p->block_size);
    w.Nkv = ceil_div(p->Lkv, p->block_size);
    w.group = p->H / p->Hkv;
    w.words = ceil_div(w.Nkv, 32);
    w.row_words = ceil_div(w.Nq, 32);
    const size_t lists = (size_t)p->B * p->H * w.Nq;
    size_t c = 0;
    if (!backward && (p->as_listed || selected_few_rows(p))) {       // needs none
        w.total = 256;
        return w;
    }
    w.index = c; c = align_up(c + lists * p->index_stride * sizeof(int32_t), 256);
    w.num = c; c = align_up(c + lists * sizeof(int32_t), 256);
    if (selected_ordered(p, w)) w.q_order = c, c = align_up(c + lists * sizeof(int32_t), 256);
    if (backward) {
        w.rows = c; c = align_up(c + (size_t)p->B * p->H * w.Nkv * w.row_words * sizeof(uint32_t), 256);
        w.counters = c; c += SELECTED_COUNTERS;
        if (selected_ordered(p, w)) {
            w.k_order = c; c = align_up(c + (size_t)p->B * p->Hkv * w.Nkv * sizeof(int32_t), 256);
        }
        w.stats = c; c = align_up(c + (size_t)p->B * p->H * selected_stats_rows(p, w.Nq) * 2 * sizeof(float), 256);
    }
    w.tuned = c;
    if (!backward && selected_sm100_forward_supported(p)) c = align_up(c + selected_sm100_forward_bytes(p), 256);
    w.total = c;
    return w;
}

static int selected_check(const wa_selected_params *p, bool backward, const char *what) {
    WA_REQUIRE(p, WA_ERR_ARG, "%s: null pointer", what);
    WA_REQUIRE(p->B > 0 && p->H > 0 && p->Hkv > 0 && p->D > 0 && p->Lq > 0 && p->Lkv > 0 && p->block_size > 0 && p->index_stride > 0, WA_ERR_ARG,
               "%s: sizes must be positive", what);
    WA_REQUIRE(p->H % p->Hkv == 0, WA_ERR_ARG, "%s: %d query heads do not divide among %d key heads", what, p->H, p->Hkv);
    WA_REQUIRE(p->D <= 256, WA_ERR_UNSUPPORTED, "%s: head_dim %d > 256", what, p->D);
    WA_REQUIRE(p->H <= 65535 && p->B <= 65535, WA_ERR_UNSUPPORTED, "%s: grid too large", what);
    WA_REQUIRE(ceil_div(p->Lkv, p->block_size) <= 32 * 48 * 1024, WA_ERR_UNSUPPORTED, "%s: more than %d key blocks", what, 32 * 48 * 1024);
    WA_REQUIRE((long long)p->Lq + 2ll * p->block_size < (1ll << 31) && (long long)p->Lkv + 2ll * p->block_size < (1ll << 31), WA_ERR_UNSUPPORTED,
               "%s: too many tokens", what);
    const wa_tensor4 *all[] = {&p->q, &p->k, &p->v, &p->out, &p->dout, &p->dq, &p->dk, &p->dv};
    const char *names[] = {"q", "k", "v", "out", "dout", "dq", "dk", "dv"};
    for (int i = 0; i < (backward ? 8 : 4); ++i) {
        WA_REQUIRE(all[i]->ptr, WA_ERR_ARG, "%s: %s is null", what, names[i]);
        WA_REQUIRE(valid_dtype(all[i]->dtype) && all[i]->dtype == p->q.dtype, WA_ERR_ARG, "%s: %s has dtype %d, q has %d", what, names[i], all[i]->dtype, p->q.dtype);
    }
    WA_REQUIRE(p->index && p->num, WA_ERR_ARG, "%s: index / num is null", what);
    WA_REQUIRE(p->lse || !backward, WA_ERR_ARG, "%s: lse is null", what);
    return 0;
}

// blocks of the queries, and for the gradient those of the keys, heaviest first
static int selected_order(const wa_selected_params *p, const SelectedPlan &w, bool backward, char *ws, cudaStream_t stream, const char *what) {
    const cudaError_t e = launch_dependent(selected_order_kernel, dim3(backward ? 2 : 1), dim3(1024), 0, stream, (const int32_t *)(ws + w.num),
                                           (const uint32_t *)(ws + w.rows), p->B * p->H * w.Nq, p->B * p->Hkv * w.Nkv, w.group * w.row_words, w.Nkv,
                                           w.group * w.Nq, (int32_t *)(ws + w.q_order), (int32_t *)(ws + w.k_order));
    if (e != cudaSuccess) return fail((int)e, "%s: %s", what, cudaGetErrorString(e));
    return check_launch(what);
}

static SelectedLists selected_lists(const wa_selected_params *p, const SelectedPlan &w, bool backward, char *ws) {
    SelectedLists l{};
    l.index = p->index; l.num = p->num; l.sizes = p->block_sizes;
    l.lists = (long long)p->B * p->H * w.Nq;
    l.Nq = w.Nq; l.Nkv = w.Nkv; l.stride = p->index_stride; l.H = p->H; l.group = w.group; l.words = w.words; l.row_words = w.row_words;
    l.warps = w.words <= SL_WORDS ? SL_WARPS : 1;
    l.as_listed = p->as_listed;
    l.clean = (int32_t *)(ws + w.index); l.clean_num = (int32_t *)(ws + w.num);
    l.rows = backward ? (uint32_t *)(ws + w.rows) : nullptr;
    return l;
}

static int launch_lists(const SelectedLists &l, cudaStream_t stream, const char *what) {
    const size_t smem = (size_t)l.warps * l.words * sizeof(uint32_t);
    static PerDeviceOnce attr_set;
    if (smem > 48 * 1024 && !attr_set.done()) {
        const cudaError_t e = cudaFuncSetAttribute(selected_lists_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 192 * 1024);
        if (e != cudaSuccess) return fail((int)e, "%s: %s", what, cudaGetErrorString(e));
        attr_set.mark();
    }
    const long long ctas = (l.lists + l.warps - 1) / l.warps;
    WA_REQUIRE(ctas < (1ll << 31), WA_ERR_UNSUPPORTED, "%s: too many query blocks", what);
    const cudaError_t e = launch_dependent(selected_lists_kernel, dim3((unsigned)ctas), dim3(l.warps * 32), smem, stream, l);
    if (e != cudaSuccess) return fail((int)e, "%s: %s", what, cudaGetErrorString(e));
    return check_launch(what);
}

static bool whole_pieces(const wa_tensor4 &t) {      // float32 rows of whole 16-byte pieces
    return t.dtype == WA_F32 && (uintptr_t)t.ptr % 16 == 0 && t.stride_b % 4 == 0 && t.stride_l % 4 == 0 && t.stride_h % 4 == 0;
}

static SelectedAny selected_any(const wa_selected_params *p, const SelectedPlan &w, char *ws) {
    SelectedAny g{};
    g.q = make_view(&p->q); g.k = make_view(&p->k); g.v = make_view(&p->v);
    g.out = p->out.ptr; g.ob = p->out.stride_b; g.ol = p->out.stride_l; g.oh = p->out.stride_h;
    g.lse = p->lse;
    g.dtype = p->q.dtype;
    g.H = p->H; g.group = w.group; g.Lq = p->Lq; g.Lkv = p->Lkv; g.D = p->D; g.block = p->block_size; g.stride = p->index_stride; g.Nq = w.Nq; g.Nkv = w.Nkv;
    g.index = (const int32_t *)(ws + w.index); g.num = (const int32_t *)(ws + w.num); g.block_sizes = p->block_sizes;
    g.scale = (float)(1.0 / sqrt((double)p->D));
    g.as_listed = p->as_listed;
    g.async = p->D % 4 == 0 && whole_pieces(p->q) && whole_pieces(p->k) && whole_pieces(p->v);
    return g;
}

}  // namespace wa

using namespace wa;

extern "C" size_t wa_selected_params_size(void) { return sizeof(wa_selected_params); }

extern "C" size_t wa_selected_workspace_bytes(const wa_selected_params *p, int backward) {
    return selected_check(p, backward != 0, "wa_selected_workspace_bytes") ? 0 : selected_plan(p, backward != 0).total;
}

extern "C" int wa_selected_forward(const wa_selected_params *p, void *stream_) {
    const char *what = "wa_selected_forward";
    const cudaStream_t stream = (cudaStream_t)stream_;
    int rc = selected_check(p, false, what);
    if (rc) return rc;
    const SelectedPlan w = selected_plan(p, false);
    WA_REQUIRE(p->workspace && p->workspace_bytes >= w.total, WA_ERR_WORKSPACE, "%s: needs a workspace of %zu bytes, got %zu", what, w.total, p->workspace_bytes);
    WA_REQUIRE((uintptr_t)p->workspace % 256 == 0, WA_ERR_ALIGN, "%s: the workspace must be 256-byte aligned", what);
    if (p->as_listed)
        return block_sparse_run(&p->q, &p->k, &p->v, &p->out, p->B, p->H, p->Lq, p->Lkv, p->D, p->block_size, p->index, p->num, p->index_stride, p->block_sizes, 0, 0,
                                p->lse, nullptr, false, stream, w.group, true);
    if (selected_few_rows(p)) return launch_few_rows(p, stream);
    char *ws = (char *)p->workspace;
    int32_t *index = (int32_t *)(ws + w.index), *num = (int32_t *)(ws + w.num);
    const bool tuned = selected_sm100_forward_supported(p);
    if (tuned && selected_sm100_cleans(p)) return selected_sm100_forward(p, p->index, p->num, num, ws + w.tuned, stream);
    if ((rc = launch_lists(selected_lists(p, w, false, ws), stream, what))) return rc;
    if (tuned) return selected_sm100_forward(p, index, num, nullptr, ws + w.tuned, stream);
    const bool ordered = selected_ordered(p, w);
    if (ordered && (rc = selected_order(p, w, false, ws, stream, what))) return rc;
    const int32_t *order = ordered ? (const int32_t *)(ws + w.q_order) : nullptr;
    // (With block sizes the kernels and the bits of wa_block_sparse_forward.  Without, it keeps bf16 with head_dim 128, which has matrix instructions there; float32 with
    // that head_dim, there -> here: 12 heads of 1170 tokens 71 -> 61 us, 64 queries over 10 blocks 109 -> 51.)
    if (!p->block_sizes && (p->D != 128 || p->q.dtype == WA_F32)) {
        SelectedAny g = selected_any(p, w, ws);
        g.q_order = order;
        return run_any<SG_FORWARD>(g, p->B, stream, what);
    }
    return block_sparse_run(&p->q, &p->k, &p->v, &p->out, p->B, p->H, p->Lq, p->Lkv, p->D, p->block_size, index, num, p->index_stride, p->block_sizes, 0, 0,
                            p->lse, order, false, stream, w.group, true);
}

extern "C" int wa_selected_backward(const wa_selected_params *p, void *stream_) {
    const char *what = "wa_selected_backward";
    const cudaStream_t stream = (cudaStream_t)stream_;
    int rc = selected_check(p, true, what);
    if (rc) return rc;
    const SelectedPlan w = selected_plan(p, true);
    WA_REQUIRE(p->workspace && p->workspace_bytes >= w.total, WA_ERR_WORKSPACE, "%s: needs a workspace of %zu bytes, got %zu", what, w.total, p->workspace_bytes);
    WA_REQUIRE((uintptr_t)p->workspace % 256 == 0, WA_ERR_ALIGN, "%s: the workspace must be 256-byte aligned", what);
    char *ws = (char *)p->workspace;
    if ((rc = launch_zeros(ws + w.rows, w.counters + SELECTED_COUNTERS - w.rows, stream, what))) return rc;
    const int32_t *index = (const int32_t *)(ws + w.index), *num = (const int32_t *)(ws + w.num);
    const uint32_t *rows = (const uint32_t *)(ws + w.rows);
    float *stats = (float *)(ws + w.stats);
    const size_t stats_rows = selected_stats_rows(p, w.Nq);
    WA_REQUIRE(stats_rows < (1ull << 31), WA_ERR_UNSUPPORTED, "%s: too many tokens", what);
    const int padded = (int)stats_rows;
    const SelectedLists lists = selected_lists(p, w, true, ws);
    if ((rc = p->q.dtype == WA_BF16 ? launch_prepare<__nv_bfloat16>(p, lists, padded, stats, stream) : launch_prepare<float>(p, lists, padded, stats, stream))) return rc;
    // dQ does not wait for dK and dV: what both read was there before the first CTA for keys let the second launch go, and its CTAs take the SMs that the
    // last ones for keys no longer need.  It ends, as the stream sees it, behind both: its CTAs wait for the first launch before they leave.
    int32_t *q_order = nullptr, *k_order = nullptr;
    if (selected_ordered(p, w)) {
        q_order = (int32_t *)(ws + w.q_order);
        k_order = (int32_t *)(ws + w.k_order);
        if ((rc = selected_order(p, w, true, ws, stream, what))) return rc;
    }
    if (selected_sm100_backward_supported(p)) return selected_sm100_backward(p, index, num, rows, stats, q_order, k_order, (int *)(ws + w.counters), stream);
    SelectedAny g = selected_any(p, w, ws);
    g.dout = make_view(&p->dout);
    g.dq = p->dq.ptr; g.dqb = p->dq.stride_b; g.dql = p->dq.stride_l; g.dqh = p->dq.stride_h;
    g.dk = p->dk.ptr; g.dkb = p->dk.stride_b; g.dkl = p->dk.stride_l; g.dkh = p->dk.stride_h;
    g.dv = p->dv.ptr; g.dvb = p->dv.stride_b; g.dvl = p->dv.stride_l; g.dvh = p->dv.stride_h;
    g.row_words = w.row_words; g.padded = padded;
    g.rows = rows; g.stats = stats; g.q_order = q_order; g.k_order = k_order;
    g.async = g.async && whole_pieces(p->dout);
    if ((rc = run_any<SG_KEYS>(g, p->B, stream, what))) return rc;
    return run_any<SG_QUERIES>(g, p->B, stream, what);
}
