// Attention over selected key blocks with its gradient: entry points, the preparation of the lists, the form for a few query rows, and the
// gradient for every shape that the tensor-core kernels (wa_hsa_sm100.cu, wa_selected_sm100.cu) do not cover.
//
// Stands in for the autograd function of wan/modules/hsa/block_sparse_triton.py:142-382.  Its dQ kernel walks the query blocks and its dK/dV
// kernel the key blocks; so do these, so that every gradient is a sum in a fixed order in one CTA's registers and nothing is added
// atomically.  The price is that scores and dP are computed twice (seven products instead of five).
#include "wa_selected.cuh"

namespace wa {

// ---- lists ---------------------------------------------------------------------------------------
// A warp per list: ids outside the key blocks and repeated ones are dropped, the others keep their order (a router's best block
// first).  For the gradient the same ids turned around: bit i of `rows` of a key block says that query block i lists it.  Bits are set
// atomically, which is the same in any order.
constexpr int SL_WARPS = 8, SL_WORDS = 1024;   // lists of a CTA; words of a bitmap up to which it has so many (32 768 key blocks)

__global__ void __launch_bounds__(SL_WARPS * 32)
selected_lists_kernel(const int32_t *__restrict__ index, const int32_t *__restrict__ num, long long lists, int Nq, int Nkv, int stride, int H, int group,
                      int words, int row_words, int32_t *__restrict__ clean, int32_t *__restrict__ clean_num, uint32_t *__restrict__ rows) {
    extern __shared__ uint32_t sl_bits[];
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long list = (long long)blockIdx.x * (blockDim.x >> 5) + warp;
    if (list >= lists) return;
    uint32_t *bits = sl_bits + (size_t)warp * words;
    for (int w = lane; w < words; w += 32) bits[w] = 0u;
    __syncwarp();
    const int n = max(0, min(num[list], stride));
    const long long bh = list / Nq;
    const int i = (int)(list - bh * Nq), h = (int)(bh % H), hh = h % group;
    const long long bhk = bh / H * (H / group) + h / group;
    int at = 0;
    for (int c = 0; c < n; c += 32) {
        const int id = c + lane < n ? index[list * stride + c + lane] : -1;
        const bool there = (unsigned)id < (unsigned)Nkv;
        const unsigned same = __match_any_sync(0xffffffffu, there ? id : -1 - lane);
        const bool take = there && lane == __ffs(same) - 1 && !((bits[id >> 5] >> (id & 31)) & 1u);
        __syncwarp();
        const unsigned all = __ballot_sync(0xffffffffu, take);
        if (take) {
            clean[list * stride + at + __popc(all & ((1u << lane) - 1u))] = id;
            atomicOr(&bits[id >> 5], 1u << (id & 31));
            if (rows) atomicOr(&rows[((bhk * Nkv + id) * group + hh) * row_words + (i >> 5)], 1u << (i & 31));
        }
        at += __popc(all);
        __syncwarp();
    }
    if (lane == 0) clean_num[list] = at;
}

// ---- row statistics of the gradient -----------------------------------------------------------------
// See selected_stat.  Reads dout and out once: `LANES` lanes take a row, 16 bytes each (LANES = 0: a warp, one channel at a time, any layout), and
// four rows are on their way at a time.
template <typename T, int LANES>
__global__ void __launch_bounds__(256)
selected_stats_kernel(View4 out, View4 dout, const float *__restrict__ lse, int H, int Lq, int D, int padded, long long all, float *__restrict__ stats) {
    constexpr int WIDE = LANES ? LANES : 32, AT_ONCE = LANES ? 4 : 1, N = 16 / sizeof(T), EACH = 256 / WIDE;
    pdl_wait();
    const int sub = threadIdx.x / WIDE, lane = threadIdx.x % WIDE;
    long long row[AT_ONCE];                       // (b, token, h), heads innermost as in memory
    long long b[AT_ONCE];
    int h[AT_ONCE], l[AT_ONCE];
    float sum[AT_ONCE], natural[AT_ONCE];
    uint4 x[AT_ONCE], y[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
        row[u] = ((long long)blockIdx.x * AT_ONCE + u) * EACH + sub;
        const long long token = row[u] / H;
        h[u] = (int)(row[u] - token * H);
        b[u] = token / padded;
        l[u] = (int)(token - b[u] * padded);
        sum[u] = 0.f;
        if (row[u] >= all || l[u] >= Lq) continue;
        natural[u] = __ldg(lse + (b[u] * H + h[u]) * Lq + l[u]);
        const T *o = (const T *)out.ptr + b[u] * out.sb + (long long)l[u] * out.sl + (long long)h[u] * out.sh;
        const T *g = (const T *)dout.ptr + b[u] * dout.sb + (long long)l[u] * dout.sl + (long long)h[u] * dout.sh;
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
            float *to = stats + (b[u] * H + h[u]) * padded * 2 + selected_stat(l[u]);
            to[0] = seen ? -1.4426950408889634f * natural[u] : -INFINITY;
            to[64] = seen ? sum[u] : 0.f;
        }
    }
}

template <typename T>
static int launch_stats(const wa_selected_params *p, int padded, float *stats, cudaStream_t stream) {
    const char *what = "wa_selected_backward";
    const auto pieces = [](const wa_tensor4 &t) {       // rows of whole 16-byte pieces
        constexpr int n = 16 / sizeof(T);
        return (uintptr_t)t.ptr % 16 == 0 && t.stride_b % n == 0 && t.stride_l % n == 0 && t.stride_h % n == 0;
    };
    const int bytes = p->D * (int)sizeof(T), lanes = pieces(p->out) && pieces(p->dout) && (bytes == 512 || bytes == 256 || bytes == 128) ? bytes / 16 : 0;
    const long long all = (long long)p->B * p->H * padded, each = lanes ? 4 * (256 / lanes) : 8, ctas = (all + each - 1) / each;
    WA_REQUIRE(ctas < (1ll << 31), WA_ERR_UNSUPPORTED, "%s: too many tokens", what);
    const auto kernel = lanes == 32 ? selected_stats_kernel<T, 32> : lanes == 16 ? selected_stats_kernel<T, 16> : lanes == 8 ? selected_stats_kernel<T, 8> : selected_stats_kernel<T, 0>;
    const cudaError_t e = launch_dependent(kernel, dim3((unsigned)ctas), dim3(256), 0, stream, make_view(&p->out), make_view(&p->dout), p->lse, p->H, p->Lq, p->D, padded, all, stats);
    if (e != cudaSuccess) return fail((int)e, "%s: %s", what, cudaGetErrorString(e));
    return check_launch(what);
}

// ---- gradient, any shape ------------------------------------------------------------------------------
// One CTA owns T rows of one side -- dQ: queries, dK/dV: keys -- and meets the rows of the other side T at a time: T x T scores and
// dP from shared memory, P and dS back to shared memory, and from there into the owned rows' sums in registers.  256 threads, 4 x 4
// (T = 64) or 2 x 2 (T = 32, head_dim above 128) of the T x T and as many owned rows by 4 * NM columns of the sums; all reads are 16 bytes.
struct SelectedGrad {
    View4 q, k, v, dout;
    void *dq, *dk, *dv;
    int dtype;
    long long dqb, dql, dqh, dkb, dkl, dkh, dvb, dvl, dvh;
    int H, group, Lq, Lkv, D, block, stride, Nq, Nkv, row_words, padded, tiles;
    const int32_t *index, *num, *block_sizes;
    const uint32_t *rows;
    const float *stats;
    float scale;
};

template <int T, int NM, bool KEYS>      // NM: 64-column steps of head_dim
__global__ void __launch_bounds__(256)
selected_grad_kernel(const SelectedGrad p) {
    constexpr int W = 64 * NM, LD = W + 4, R = T / 16, LP = T + 4;
    extern __shared__ __align__(16) float sg_smem[];
    float *f1 = sg_smem, *f2 = f1 + T * LD, *g1 = f2 + T * LD, *g2 = g1 + T * LD;      // owned: q, dout or k, v; met: the other two
    float *ps = g2 + T * LD, *ds = ps + T * LP;
    float2 *st = reinterpret_cast<float2 *>(ds + T * LP);                               // statistics of the T query rows
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int blk = blockIdx.x / p.tiles, first = blk * p.block + (blockIdx.x % p.tiles) * T, b = blockIdx.z;
    const int hk = KEYS ? blockIdx.y : blockIdx.y / p.group;
    const auto keys_of = [&](int id) {       // real tokens of a key block
        const int n = min(p.block, p.Lkv - id * p.block);
        return p.block_sizes ? max(0, min(n, p.block_sizes[id])) : n;
    };
    const int own_end = min(min(first + T, (blk + 1) * p.block), KEYS ? p.Lkv : p.Lq);       // rows to write
    const int own_real = KEYS ? min(own_end, blk * p.block + keys_of(blk)) : own_end;         // rows that count
    if (first >= own_end) return;

    const auto bring = [&](float *to, const View4 &x, int h, int from, int end) {
        const long long base = b * x.sb + (long long)h * x.sh;
        for (int e = threadIdx.x; e < T * W; e += 256) {
            const int r = e / W, d = e % W;
            to[r * LD + d] = from + r < end && d < p.D ? load_elem(x.ptr, x.dtype, base + (long long)(from + r) * x.sl + d) : 0.f;
        }
    };
    const auto bring_stats = [&](int h, int from, int end) {
        const float *stats = p.stats + ((long long)b * p.H + h) * p.padded * 2;
        for (int r = threadIdx.x; r < T; r += 256)
            st[r] = from + r < end ? make_float2(stats[selected_stat(from + r)], stats[selected_stat(from + r) + 64]) : make_float2(-INFINITY, 0.f);
    };
    bring(f1, KEYS ? p.k : p.q, KEYS ? hk : blockIdx.y, first, own_real);
    bring(f2, KEYS ? p.v : p.dout, KEYS ? hk : blockIdx.y, first, own_real);
    if (!KEYS) bring_stats(blockIdx.y, first, own_real);

    float4 sum1[R][NM], sum2[R][NM];         // of the owned rows: dV (KEYS), dK or dQ
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int m = 0; m < NM; ++m) sum1[i][m] = sum2[i][m] = make_float4(0.f, 0.f, 0.f, 0.f);
    const float to_log2 = p.scale * 1.4426950408889634f;
    const int depth = (p.D + 3) & ~3;

    const auto meet = [&](int h, int from, int end) {       // rows from .. end of the other side
        __syncthreads();
        bring(g1, KEYS ? p.q : p.k, KEYS ? h : hk, from, end);
        bring(g2, KEYS ? p.dout : p.v, KEYS ? h : hk, from, end);
        if (KEYS) bring_stats(h, from, end);
        __syncthreads();
        float s[R][R], dp[R][R];
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < R; ++j) s[i][j] = dp[i][j] = 0.f;
        const auto dots = [&](float (&acc)[R][R], const float *f, const float *g) {
            for (int d = 0; d < depth; d += 4) {
                float4 x[R], y[R];
#pragma unroll
                for (int i = 0; i < R; ++i) x[i] = *reinterpret_cast<const float4 *>(f + (ty * R + i) * LD + d);
#pragma unroll
                for (int j = 0; j < R; ++j) y[j] = *reinterpret_cast<const float4 *>(g + (tx + 16 * j) * LD + d);
#pragma unroll
                for (int i = 0; i < R; ++i)
#pragma unroll
                    for (int j = 0; j < R; ++j) {
                        acc[i][j] = fmaf(x[i].x, y[j].x, acc[i][j]);
                        acc[i][j] = fmaf(x[i].y, y[j].y, acc[i][j]);
                        acc[i][j] = fmaf(x[i].z, y[j].z, acc[i][j]);
                        acc[i][j] = fmaf(x[i].w, y[j].w, acc[i][j]);
                    }
            }
        };
        dots(s, f1, g1);
        dots(dp, f2, g2);
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < R; ++j) {
                const int f = ty * R + i, g = tx + 16 * j;
                const float2 row = st[KEYS ? g : f];
                const bool there = first + f < own_real && from + g < end;
                const float pr = there ? exp2f(fmaf(s[i][j], to_log2, row.x)) : 0.f;
                ps[f * LP + g] = pr;
                ds[f * LP + g] = there ? pr * (dp[i][j] - row.y) * p.scale : 0.f;
            }
        __syncthreads();
        const auto add = [&](float4 (&acc)[R][NM], const float *w, const float *x) {
            for (int g = 0; g < T; g += 4) {
                float4 a[R];
#pragma unroll
                for (int i = 0; i < R; ++i) a[i] = *reinterpret_cast<const float4 *>(w + (ty * R + i) * LP + g);
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int m = 0; m < NM; ++m) {
                        const float4 y = *reinterpret_cast<const float4 *>(x + (g + u) * LD + 64 * m + 4 * tx);
#pragma unroll
                        for (int i = 0; i < R; ++i) {
                            const float c = u == 0 ? a[i].x : u == 1 ? a[i].y : u == 2 ? a[i].z : a[i].w;
                            acc[i][m].x = fmaf(c, y.x, acc[i][m].x);
                            acc[i][m].y = fmaf(c, y.y, acc[i][m].y);
                            acc[i][m].z = fmaf(c, y.z, acc[i][m].z);
                            acc[i][m].w = fmaf(c, y.w, acc[i][m].w);
                        }
                    }
            }
        };
        if (KEYS) add(sum1, ps, g2);
        add(sum2, ds, g1);
    };
    if (KEYS) {
        const uint32_t *bits = p.rows + (((long long)b * (p.H / p.group) + hk) * p.Nkv + blk) * p.group * p.row_words;
        for (int w = 0; w < p.group * p.row_words; ++w)
            for (uint32_t left = bits[w]; left; left &= left - 1) {
                const int i = (w % p.row_words) * 32 + __ffs(left) - 1, end = min((i + 1) * p.block, p.Lq);
                for (int from = i * p.block; from < end; from += T) meet(hk * p.group + w / p.row_words, from, min(from + T, end));
            }
    } else {
        const long long list = ((long long)b * p.H + blockIdx.y) * p.Nq + blk;
        for (int n = 0; n < p.num[list]; ++n) {
            const int id = p.index[list * p.stride + n], end = id * p.block + keys_of(id);
            for (int from = id * p.block; from < end; from += T) meet(blockIdx.y, from, min(from + T, end));
        }
    }
    const auto write = [&](const float4 (&acc)[R][NM], void *to, long long sb, long long sl, int h, long long sh) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int r = first + ty * R + i;
            if (r >= own_end) continue;
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                const float v[4] = {acc[i][m].x, acc[i][m].y, acc[i][m].z, acc[i][m].w};
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (64 * m + 4 * tx + u < p.D) store_elem(to, p.dtype, b * sb + r * sl + h * sh + 64 * m + 4 * tx + u, v[u]);
            }
        }
    };
    if (KEYS) {
        write(sum1, p.dv, p.dvb, p.dvl, hk, p.dvh);
        write(sum2, p.dk, p.dkb, p.dkl, hk, p.dkh);
    } else {
        write(sum2, p.dq, p.dqb, p.dql, blockIdx.y, p.dqh);
    }
}

template <int T, int NM>
static int launch_grad(SelectedGrad p, int B, int Hkv, cudaStream_t stream) {
    const char *what = "wa_selected_backward";
    constexpr size_t smem = (size_t)(4 * T * (64 * NM + 4) + 2 * T * (T + 4)) * 4 + T * 8;
    static PerDeviceOnce attr_set;
    if (!attr_set.done()) {
        cudaError_t e = cudaFuncSetAttribute(selected_grad_kernel<T, NM, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(selected_grad_kernel<T, NM, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return fail((int)e, "%s: %s", what, cudaGetErrorString(e));
        attr_set.mark();
    }
    p.tiles = ceil_div(p.block, T);
    const long long kx = (long long)p.Nkv * p.tiles, qx = (long long)p.Nq * p.tiles;
    WA_REQUIRE(kx < (1ll << 31) && qx < (1ll << 31), WA_ERR_UNSUPPORTED, "%s: grid too large", what);
    int rc;
    selected_grad_kernel<T, NM, true><<<dim3((unsigned)kx, Hkv, B), 256, smem, stream>>>(p);
    if ((rc = check_launch(what))) return rc;
    selected_grad_kernel<T, NM, false><<<dim3((unsigned)qx, p.H, B), 256, smem, stream>>>(p);
    return check_launch(what);
}

// ---- host ----------------------------------------------------------------------------------------
static SelectedPlan selected_plan(const wa_selected_params *p, bool backward) {
    SelectedPlan w{};
    w.Nq = ceil_div(p->Lq, p->block_size);
    w.Nkv = ceil_div(p->Lkv, p->block_size);
    w.group = p->H / p->Hkv;
    w.words = ceil_div(w.Nkv, 32);
    w.row_words = ceil_div(w.Nq, 32);
    const size_t lists = (size_t)p->B * p->H * w.Nq;
    size_t c = 0;
    w.index = c; c = align_up(c + lists * p->index_stride * sizeof(int32_t), 256);
    w.num = c; c = align_up(c + lists * sizeof(int32_t), 256);
    if (backward) {
        w.rows = c; c = align_up(c + (size_t)p->B * p->H * w.Nkv * w.row_words * sizeof(uint32_t), 256);
        w.stats = c; c = align_up(c + (size_t)p->B * p->H * selected_stats_rows(p, w.Nq) * 2 * sizeof(float), 256);
    }
    w.tuned = c;
    if (backward ? selected_sm100_backward_supported(p) : selected_sm100_forward_supported(p))
        c = align_up(c + (backward ? selected_sm100_backward_bytes(p) : selected_sm100_forward_bytes(p)), 256);
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

static int selected_lists(const wa_selected_params *p, const SelectedPlan &w, bool backward, char *ws, cudaStream_t stream, const char *what) {
    const long long lists = (long long)p->B * p->H * w.Nq;
    uint32_t *rows = backward ? (uint32_t *)(ws + w.rows) : nullptr;
    if (rows) {
        const cudaError_t e = cudaMemsetAsync(rows, 0, (size_t)p->B * p->H * w.Nkv * w.row_words * sizeof(uint32_t), stream);
        if (e != cudaSuccess) return fail((int)e, "%s: %s", what, cudaGetErrorString(e));
    }
    const int warps = w.words <= SL_WORDS ? SL_WARPS : 1;
    const size_t smem = (size_t)warps * w.words * sizeof(uint32_t);
    static PerDeviceOnce attr_set;
    if (smem > 48 * 1024 && !attr_set.done()) {
        const cudaError_t e = cudaFuncSetAttribute(selected_lists_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 192 * 1024);
        if (e != cudaSuccess) return fail((int)e, "%s: %s", what, cudaGetErrorString(e));
        attr_set.mark();
    }
    const long long ctas = (lists + warps - 1) / warps;
    WA_REQUIRE(ctas < (1ll << 31), WA_ERR_UNSUPPORTED, "%s: too many query blocks", what);
    const cudaError_t e = launch_dependent(selected_lists_kernel, dim3((unsigned)ctas), dim3(warps * 32), smem, stream, p->index, p->num, lists, w.Nq, w.Nkv,
                                           p->index_stride, p->H, w.group, w.words, w.row_words, (int32_t *)(ws + w.index), (int32_t *)(ws + w.num), rows);
    if (e != cudaSuccess) return fail((int)e, "%s: %s", what, cudaGetErrorString(e));
    return check_launch(what);
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
    char *ws = (char *)p->workspace;
    if ((rc = selected_lists(p, w, false, ws, stream, what))) return rc;
    const int32_t *index = (const int32_t *)(ws + w.index), *num = (const int32_t *)(ws + w.num);
    if (selected_sm100_forward_supported(p)) return selected_sm100_forward(p, index, num, ws + w.tuned, stream);
    return block_sparse_run(&p->q, &p->k, &p->v, &p->out, p->B, p->H, p->Lq, p->Lkv, p->D, p->block_size, index, num, p->index_stride, p->block_sizes, 0, 0,
                            p->lse, nullptr, false, stream, w.group);
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
    if ((rc = selected_lists(p, w, true, ws, stream, what))) return rc;
    const int32_t *index = (const int32_t *)(ws + w.index), *num = (const int32_t *)(ws + w.num);
    const uint32_t *rows = (const uint32_t *)(ws + w.rows);
    float *stats = (float *)(ws + w.stats);
    const size_t stats_rows = selected_stats_rows(p, w.Nq);
    WA_REQUIRE(stats_rows < (1ull << 31), WA_ERR_UNSUPPORTED, "%s: too many tokens", what);
    const int padded = (int)stats_rows;
    if ((rc = p->q.dtype == WA_BF16 ? launch_stats<__nv_bfloat16>(p, padded, stats, stream) : launch_stats<float>(p, padded, stats, stream))) return rc;
    if (selected_sm100_backward_supported(p)) return selected_sm100_backward(p, index, num, rows, stats, ws + w.tuned, stream);
    SelectedGrad g{};
    g.q = make_view(&p->q); g.k = make_view(&p->k); g.v = make_view(&p->v); g.dout = make_view(&p->dout);
    g.dq = p->dq.ptr; g.dqb = p->dq.stride_b; g.dql = p->dq.stride_l; g.dqh = p->dq.stride_h;
    g.dk = p->dk.ptr; g.dkb = p->dk.stride_b; g.dkl = p->dk.stride_l; g.dkh = p->dk.stride_h;
    g.dv = p->dv.ptr; g.dvb = p->dv.stride_b; g.dvl = p->dv.stride_l; g.dvh = p->dv.stride_h;
    g.dtype = p->q.dtype;
    g.H = p->H; g.group = w.group; g.Lq = p->Lq; g.Lkv = p->Lkv; g.D = p->D; g.block = p->block_size; g.stride = p->index_stride;
    g.Nq = w.Nq; g.Nkv = w.Nkv; g.row_words = w.row_words; g.padded = padded;
    g.index = index; g.num = num; g.block_sizes = p->block_sizes; g.rows = rows; g.stats = stats;
    g.scale = (float)(1.0 / sqrt((double)p->D));
    if (p->D <= 64) return launch_grad<64, 1>(g, p->B, p->Hkv, stream);
    if (p->D <= 128) return launch_grad<64, 2>(g, p->B, p->Hkv, stream);
    return launch_grad<32, 4>(g, p->B, p->Hkv, stream);
}
