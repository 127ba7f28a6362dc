// The steps of a latent-attention layer around the attention itself:
//   vib3_launch_latent_append_paged   normalise, rotate and store a step's rows into the paged cache
//   vib3_launch_latent_query          per head q_nope . W_uk and the rotation of q_rope
//   vib3_launch_latent_value          per head o . W_uv^T
// The reference has a scalar kernel for each (vib3_mla_kv_cache_append_kernel, vib3_mla_q_absorb_rope_kernel,
// vib3_mla_v_reconstruct, cuda/src/kernels.cu:1709, :1679, :1624), for one token and a flat cache.
#include "latent_tc.cuh"

namespace vib3 {

// ── append ───────────────────────────────────────────────────────────────────────────────────
// row[0:512] = x / sqrt(mean(x^2) + eps) * w, row[512:576] = rotated x, rounded once.  One warp per token: the row stays in
// registers between the sum of squares and the scaling, so a token is read once and written once.  Bound by the launch for a
// decode step (29 tokens 1.8 us), by HBM for a prompt (8191 tokens 4.9 us, 5.8 TB/s).
struct AppendArgs {
    const void* x;
    long long x_stride;   // elements
    const void* norm;     // cache's type, or null
    float eps;
    const int* positions;
    const long long* slots;
    const double* inv_freq;
    float rope_scale;
    int pairs, n_tokens;
    void* cache;
    long long n_slots;
    int page_size;
    long long page_stride, row_stride;   // elements
    int* status;
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float* v) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        const T* t = reinterpret_cast<const T*>(&a);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = as_float(t[i]);
    }
}

constexpr int kAppendWarps = 4;

template <typename TX, typename TC>
__global__ void __launch_bounds__(kAppendWarps * 32) latent_append_kernel(AppendArgs a) {
    pdl_enter();
    const int lane = threadIdx.x & 31;
    const int t = blockIdx.x * kAppendWarps + (threadIdx.x >> 5);
    if (t >= a.n_tokens) return;
    const long long slot = a.slots[t];
    if (slot < 0) return;   // a padding token
    if (slot >= a.n_slots) {
        if (lane == 0 && a.status) atomicOr(a.status, kStatusBadPage);
        return;
    }
    const TX* x = reinterpret_cast<const TX*>(a.x) + t * a.x_stride;
    TC* row = reinterpret_cast<TC*>(a.cache) + (slot / a.page_size) * a.page_stride + (slot % a.page_size) * a.row_stride;
    float v[2][8];
    load8(x + lane * 8, v[0]);
    load8(x + 256 + lane * 8, v[1]);
    const int i0 = a.pairs ? 2 * lane : lane, i1 = a.pairs ? 2 * lane + 1 : lane + 32;
    const float p = as_float(x[kRank + i0]), q = as_float(x[kRank + i1]);
    float c, s;
    rope_angle(a.positions[t], a.inv_freq[lane], a.rope_scale, c, s);
    if (a.norm) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(v[0][i], v[0][i], fmaf(v[1][i], v[1][i], ss));
#pragma unroll
        for (int m = 16; m; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
        const float inv = 1.0f / sqrtf(ss * (1.0f / kRank) + a.eps);
        float w[8];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            load8(reinterpret_cast<const TC*>(a.norm) + j * 256 + lane * 8, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j][i] = v[j][i] * inv * w[i];
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        uint4 o;
        o.x = pack2<TC>(v[j][0], v[j][1]); o.y = pack2<TC>(v[j][2], v[j][3]);
        o.z = pack2<TC>(v[j][4], v[j][5]); o.w = pack2<TC>(v[j][6], v[j][7]);
        *reinterpret_cast<uint4*>(row + j * 256 + lane * 8) = o;
    }
    const float u = p * c - q * s, w = q * c + p * s;
    if (a.pairs) {
        *reinterpret_cast<uint32_t*>(row + kRank + i0) = pack2<TC>(u, w);
    } else {
        row[kRank + i0] = from_float<TC>(u);
        row[kRank + i1] = from_float<TC>(w);
    }
}

// ── per-head products ────────────────────────────────────────────────────────────────────────
// C[t, n] = sum_k A[t, k] B(k, n) for one head.  A tile is 128 tokens (fewer are padded) and 128 or 64 columns; A and B come as
// chunks of 64 values of K through a ring, the sum stays in tensor memory, and the rounded tile leaves through shared memory as tensor
// copies, which leave out what lies beyond the last token or column.
//   query: A = q_nope [tokens][nope], B = W_uk[h] [nope][512]: columns contiguous (MN-major)
//   value: A = o [tokens][512],       B = W_uv[h] [value][512]: K contiguous
// These products are bound by their bytes: with one token the head matrices are read for two flops per value, with 512 a query's
// result rows are most of the traffic (and the tensor pipe is busy for a fifth of the time).  So what counts is many bytes in flight
// with few instructions (warp-level MMAs fed by 16-byte copies spent their time on addresses: 500 queries of 64 heads in 32 us), and that
// reads and writes overlap: a CTA per SM takes tile after tile, the ring (160 KB) runs ahead across them, and of two accumulators one is
// stored while the other is filled.  (A CTA per tile, all of them loading and then all of them storing: 16.7 us; two CTAs per SM with a
// third of the ring each, where a tile's loads waited for the tile before: 15.8; now 13.0 us, 4.4 TB/s.)  One query or value: 3.8 and 4.7 us.
constexpr int kHeadTokens = 128, kHeadAChunk = kHeadTokens * 128, kHeadMaxStages = 12, kHeadMaxCols = 128;
constexpr int kHeadOut = kHeadTokens * kHeadMaxCols * 2, kHeadRing = 160 * 1024;   // (two such tiles)
constexpr int kHeadThreads = 320;          // copies, MMAs, four warps for the results, four for the rotation

struct HeadMaps {
    CUtensorMap a, b, c;
};

struct HeadArgs {
    const void* a;
    long long a_token, a_head;   // strides in elements
    const void* w;
    long long w_head;
    void* out;
    long long out_token, out_head;
    int n_tokens, heads, dim;    // dim: nope (query) or value width
    // the query's rotation
    const int* positions;
    const double* inv_freq;
    float rope_scale;
    int pairs;
    int* status;
    // the split
    int k_steps, n_cols, col_blocks, stages, a_rows, tiles;   // MMAs of 16 along K, columns of a tile, ..., tokens that a copy of A brings
};

constexpr int kRotateHeads = 8;    // heads that share one evaluation of a token's angles

// The 64 position values of up to eight heads of a token, by half a warp: a lane turns two pairs.
template <typename T>
__device__ __forceinline__ void rotate_heads(const HeadArgs& g, int t, int h0) {
    const int l = threadIdx.x & 15, hn = min(kRotateHeads, g.heads - h0);
    const T* q = (const T*)g.a + t * g.a_token + h0 * g.a_head + g.dim;
    T* o = (T*)g.out + t * g.out_token + h0 * g.out_head + kRank;
    // neighbours: values 4 l .. 4 l + 3; halves: 2 l, 2 l + 1 and the same 32 further
    const int x = g.pairs ? 4 * l : 2 * l, y = g.pairs ? 4 * l + 2 : 2 * l + 32;
    uint32_t u[kRotateHeads], v[kRotateHeads];
#pragma unroll
    for (int h = 0; h < kRotateHeads; ++h)
        if (h < hn) {
            u[h] = *reinterpret_cast<const uint32_t*>(q + h * g.a_head + x);
            v[h] = *reinterpret_cast<const uint32_t*>(q + h * g.a_head + y);
        }
    float c0, s0, c1, s1;
    rope_angle(g.positions[t], g.inv_freq[2 * l], g.rope_scale, c0, s0);
    rope_angle(g.positions[t], g.inv_freq[2 * l + 1], g.rope_scale, c1, s1);
#pragma unroll
    for (int h = 0; h < kRotateHeads; ++h)
        if (h < hn) {
            const float2 p = unpack2<T>(u[h]), r = unpack2<T>(v[h]);
            uint32_t a, b;
            if (g.pairs) {
                a = pack2<T>(p.x * c0 - p.y * s0, p.y * c0 + p.x * s0);
                b = pack2<T>(r.x * c1 - r.y * s1, r.y * c1 + r.x * s1);
            } else {
                a = pack2<T>(p.x * c0 - r.x * s0, p.y * c1 - r.y * s1);
                b = pack2<T>(r.x * c0 + p.x * s0, r.y * c1 + p.y * s1);
            }
            *reinterpret_cast<uint32_t*>(o + h * g.out_head + x) = a;
            *reinterpret_cast<uint32_t*>(o + h * g.out_head + y) = b;
        }
}

// Tile = (tile of tokens * heads + head) * column blocks + column block.
// (One block per SM, which its shared memory allows anyway, has to be said: the compiler otherwise keeps to 85 registers, puts fewer of the
// rotation's loads in flight, and 500 queries take 14.7 us instead of 13.2.)
template <typename T, bool QUERY>
__global__ void __launch_bounds__(kHeadThreads, 1) latent_head_kernel(const __grid_constant__ HeadMaps maps, const HeadArgs g) {
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ uint64_t full[kHeadMaxStages], empty[kHeadMaxStages], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_at;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    // (the swizzle goes by the address, and the static arrays stand before the dynamic memory)
    const uint32_t out_at = (smem_u32(smem) + 1023u) & ~1023u, base = out_at + 2 * kHeadOut;
    // (A's rows behind the copied ones are whatever lies there: the MMA reads them, and their sums are not stored)
    const uint32_t a_bytes = (uint32_t)g.a_rows * 128, b_bytes = (uint32_t)g.n_cols * 128, stage_bytes = a_bytes + b_bytes;
    const int chunks = (g.k_steps + 3) >> 2;
    const uint32_t tmem_cols = 2 * (uint32_t)g.n_cols;      // 128 or 256
    if (tid == 0) {
        for (int s = 0; s < g.stages; ++s) {
            bar_init(&full[s], 1);
            bar_init(&empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            bar_init(&acc_full[s], 1);
            bar_init(&acc_empty[s], 128);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_at)), "r"(tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = uniform(tmem_at);
    pdl_enter();
    bool ok = true;
    int s = 0;              // ring stage and the parity of its use
    unsigned parity = 0;
    auto advance = [&] {
        if (++s == g.stages) {
            s = 0;
            parity ^= 1;
        }
    };
    if (warp == 0) {
        if (elect_one()) {
            int n = 0;      // chunks so far
            for (int tile = blockIdx.x; ok && tile < g.tiles; tile += gridDim.x) {
                const int col = tile % g.col_blocks * g.n_cols, h = tile / g.col_blocks % g.heads, t0 = tile / g.col_blocks / g.heads * kHeadTokens;
                for (int c = 0; c < chunks; ++c, ++n) {
                    if (n >= g.stages && !bar_wait(&empty[s], parity ^ 1)) {
                        ok = false;
                        break;
                    }
                    const uint32_t at = base + s * stage_bytes;
                    bar_expect(&full[s], stage_bytes);
                    tma_load_3d(at, &maps.a, 64 * c, h, t0, &full[s]);
                    if (QUERY)
                        for (int x = 0; x < g.n_cols / 64; ++x) tma_load_3d(at + a_bytes + x * kChunkBytes, &maps.b, col + 64 * x, 64 * c, h, &full[s]);
                    else
                        tma_load_3d(at + a_bytes, &maps.b, 64 * c, col, h, &full[s]);
                    advance();
                }
            }
            // nothing is in flight to this CTA's memory when it leaves, neither copies nor the releases of their stages
            for (int x = n > g.stages ? n - g.stages : 0; x < n; ++x) {
                const bool in = bar_wait(&full[x % g.stages], (x / g.stages) & 1);
                ok = ok && in && bar_wait(&empty[x % g.stages], (x / g.stages) & 1);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        const uint32_t id = uniform(idesc<T>(128, (uint32_t)g.n_cols, false, QUERY));
        int i = 0;          // tiles so far
        for (int tile = blockIdx.x; ok && tile < g.tiles; tile += gridDim.x, ++i) {
            ok = i < 2 || bar_wait_warp(&acc_empty[i & 1], (unsigned)((i >> 1) - 1) & 1);
            const uint32_t d = uniform(tmem + (uint32_t)((i & 1) * g.n_cols));
            for (int c = 0; c < chunks; ++c) {
                const int steps = min(4, g.k_steps - 4 * c);
                ok = ok && bar_wait_warp(&full[s], parity);
                if (!ok) break;
                tc_fence_after();
                const uint32_t at = base + s * stage_bytes, ad = uniform(desc_k(at)), bd = uniform(QUERY ? desc_mn(at + a_bytes) : desc_k(at + a_bytes));
                if (elect_one()) {
                    for (int k = 0; k < steps; ++k) umma_ss(d, ad + k * 2, bd + k * (QUERY ? 2048 / 16 : 2), id, (uint32_t)(c + k > 0));
                    umma_commit(&empty[s]);
                    if (c == chunks - 1) umma_commit(&acc_full[i & 1]);
                }
                __syncwarp();
                advance();
            }
        }
        if (!ok) {          // what was issued has to be through before the tensor memory is freed
            if (elect_one()) umma_commit(&acc_full[i & 1]);
            __syncwarp();
            bar_wait_warp(&acc_full[i & 1], (unsigned)(i >> 1) & 1);
        }
    } else if (warp >= 6) {
        if (QUERY) {
            // The rotation beside the products: half a warp takes (token, eight heads) after (token, eight heads).  (As blocks of their own they
            // held as much shared memory as a product's; by the warps of the results, before those, four rounds of it took 10000 cycles.)
            const int groups = (g.heads + kRotateHeads - 1) / kRotateHeads;
            for (int i = blockIdx.x * 8 + ((tid - 192) >> 4); i < g.n_tokens * groups; i += gridDim.x * 8)
                rotate_heads<T>(g, i / groups, i % groups * kRotateHeads);
            __syncwarp();
        }
    } else {
        // A tile's sums to shared memory as chunks of 64 columns, the tensor copy's layout, and out.
        const int row = 32 * (warp & 3) + lane;
        int i = 0;
        for (int tile = blockIdx.x; ok && tile < g.tiles; tile += gridDim.x, ++i) {
            const int col = tile % g.col_blocks * g.n_cols, h = tile / g.col_blocks % g.heads, t0 = tile / g.col_blocks / g.heads * kHeadTokens;
            ok = bar_wait_warp(&acc_full[i & 1], (unsigned)(i >> 1) & 1);
            // (the copies of the tile two before have read their place; every warp comes to these barriers)
            if (warp == 2 && elect_one()) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
            __syncwarp();
            bool all;
            {
                uint32_t r;
                asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                             : "=r"(r) : "r"((uint32_t)ok) : "memory");
                all = r != 0;
            }
            ok = all;
            if (!ok) break;
            tc_fence_after();
            for (int x = 0; x < g.n_cols / 32; ++x) {
                uint32_t o[32];
                tmem_ld_32x32(tmem + (i & 1) * g.n_cols + 32 * x + ((uint32_t)(32 * (warp & 3)) << 16), o);
                tmem_ld_wait();
                unsigned char* to = smem + (out_at - smem_u32(smem)) + (i & 1) * kHeadOut + (x >> 1) * kHeadAChunk + row * 128;
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    uint4 b;
                    b.x = pack2<T>(__uint_as_float(o[8 * y]), __uint_as_float(o[8 * y + 1]));
                    b.y = pack2<T>(__uint_as_float(o[8 * y + 2]), __uint_as_float(o[8 * y + 3]));
                    b.z = pack2<T>(__uint_as_float(o[8 * y + 4]), __uint_as_float(o[8 * y + 5]));
                    b.w = pack2<T>(__uint_as_float(o[8 * y + 6]), __uint_as_float(o[8 * y + 7]));
                    *reinterpret_cast<uint4*>(to + ((((x & 1) * 4 + y) ^ (row & 7)) << 4)) = b;
                }
            }
            tc_fence_before();
            bar_arrive(&acc_empty[i & 1]);
            proxy_fence();
            asm volatile("bar.sync 1, 128;" ::: "memory");
            if (warp == 2 && elect_one()) {
                for (int x = 0; x < g.n_cols / 64; ++x)
                    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];"
                                 ::"l"(&maps.c), "r"(col + 64 * x), "r"(h), "r"(t0), "r"(out_at + (i & 1) * kHeadOut + x * kHeadAChunk) : "memory");
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
            __syncwarp();
        }
        if (warp == 2 && elect_one()) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
    }
    // (by every thread: in the copying warp one lane alone knows)
    if (!ok && g.status) atomicOr(g.status, kStatusTimeout);
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_cols) : "memory");
    }
}

namespace {

int ceil_div(int a, int b) { return (a + b - 1) / b; }

template <typename T, bool QUERY>
int launch_heads(HeadArgs g, int dtype, cudaStream_t st) {
    if (!tensor_map_encoder()) return VIB3_ERR_UNSUPPORTED;
    const int tiles = ceil_div(g.n_tokens, kHeadTokens), n_all = QUERY ? kRank : g.dim, k_all = QUERY ? g.dim : kRank;
    g.k_steps = k_all / 16;
    // 128 columns unless the tiles are then fewer than the SMs (wider ones read A less often).
    g.n_cols = n_all > 64 && tiles * g.heads * ceil_div(n_all, kHeadMaxCols) >= sm_count() ? kHeadMaxCols : 64;
    g.col_blocks = ceil_div(n_all, g.n_cols);
    g.tiles = tiles * g.heads * g.col_blocks;
    g.a_rows = g.n_tokens >= kHeadTokens ? kHeadTokens : ceil_div(g.n_tokens, 8) * 8;
    // Behind the ring lie the rows that an MMA of the last stage reads beyond a short A.
    const int stage = g.a_rows * 128 + g.n_cols * 128, tail = kHeadAChunk - g.a_rows * 128;
    g.stages = (kHeadRing - tail) / stage < kHeadMaxStages ? (kHeadRing - tail) / stage : kHeadMaxStages;
    const int smem = 1024 + 2 * kHeadOut + g.stages * stage + tail;
    const int e = allow_smem<latent_head_kernel<T, QUERY>>(1024 + 2 * kHeadOut + kHeadRing);
    if (e) return e;
    HeadMaps maps;
    const long long width = QUERY ? g.dim + kRope : kRank, out_width = QUERY ? kLatentRow : g.dim;
    // (a dimension of one has no stride that matters)
    const long long at = g.n_tokens > 1 ? g.a_token : width, ah = g.heads > 1 ? g.a_head : width, ot = g.n_tokens > 1 ? g.out_token : out_width,
                    oh = g.heads > 1 ? g.out_head : out_width, wh = g.heads > 1 ? g.w_head : (long long)k_all * n_all;
    if (!map_3d(&maps.a, dtype, g.a, width, g.heads, g.n_tokens, ah, at, 1, g.a_rows) ||
        !(QUERY ? map_3d(&maps.b, dtype, g.w, kRank, g.dim, g.heads, kRank, wh, 64, 1) : map_3d(&maps.b, dtype, g.w, kRank, g.dim, g.heads, kRank, wh, g.n_cols, 1)) ||
        !map_3d(&maps.c, dtype, g.out, out_width, g.heads, g.n_tokens, oh, ot, 1, kHeadTokens))
        return VIB3_ERR_SHAPE;
    return launch_latent(latent_head_kernel<T, QUERY>, dim3((unsigned)(g.tiles < sm_count() ? g.tiles : sm_count())), kHeadThreads, (size_t)smem, st, maps, g);
}

bool off16(const void* p) { return ((uintptr_t)p & 15) != 0; }

// The largest call: kernels index tokens, heads and blocks in 32 bits.
constexpr int kLatentMaxTokens = 1 << 20;

}  // namespace

}  // namespace vib3

using namespace vib3;

extern "C" int vib3_launch_latent_append_paged(const void* kv, int kv_dtype, long long kv_stride, const void* norm_weight_or_null, float eps,
                                               const int* positions, const long long* slots, const double* inv_freq, float rope_scale,
                                               int pairs, int n_tokens, void* cache, int cache_dtype, long long num_pages, int page_size,
                                               long long page_stride, long long row_stride, int* status, void* stream) {
    if ((n_tokens != 0 && (!kv || !positions || !slots)) || !inv_freq || !cache) return VIB3_ERR_NULL;     // (no tokens: an empty tensor's address is null)
    if (n_tokens < 0 || n_tokens > kLatentMaxTokens || num_pages <= 0 || page_size <= 0) return VIB3_ERR_COUNT;
    if (kv_dtype < L_F32 || kv_dtype > L_BF16 || (cache_dtype != L_F16 && cache_dtype != L_BF16)) return VIB3_ERR_UNSUPPORTED;
    const int per16 = kv_dtype == L_F32 ? 4 : 8;
    if (off16(kv) || kv_stride % per16 || off16(norm_weight_or_null) || off16(cache) || page_stride % 8 || row_stride % 8) return VIB3_ERR_ALIGN;
    if (row_stride < kLatentRow || page_stride < 0 || (num_pages > 1 && page_stride < row_stride * (page_size - 1) + kLatentRow) ||
        (n_tokens > 1 && kv_stride < kLatentRow))
        return VIB3_ERR_SHAPE;
    if (n_tokens == 0) return VIB3_OK;
    AppendArgs a{kv, kv_stride, norm_weight_or_null, eps, positions, slots, inv_freq, rope_scale, pairs, n_tokens, cache,
                 num_pages * page_size, page_size, page_stride, row_stride, status};
    const dim3 grid((unsigned)ceil_div(n_tokens, kAppendWarps));
    const int threads = kAppendWarps * 32;
    cudaStream_t st = (cudaStream_t)stream;
    if (cache_dtype == L_F16) {
        if (kv_dtype == L_F32) return launch_latent(latent_append_kernel<float, __half>, grid, threads, 0, st, a);
        if (kv_dtype == L_F16) return launch_latent(latent_append_kernel<__half, __half>, grid, threads, 0, st, a);
        return launch_latent(latent_append_kernel<__nv_bfloat16, __half>, grid, threads, 0, st, a);
    }
    if (kv_dtype == L_F32) return launch_latent(latent_append_kernel<float, __nv_bfloat16>, grid, threads, 0, st, a);
    if (kv_dtype == L_F16) return launch_latent(latent_append_kernel<__half, __nv_bfloat16>, grid, threads, 0, st, a);
    return launch_latent(latent_append_kernel<__nv_bfloat16, __nv_bfloat16>, grid, threads, 0, st, a);
}

static int check_heads(const HeadArgs& g, int dtype, int out_width) {
    if ((g.n_tokens != 0 && (!g.a || !g.out)) || !g.w) return VIB3_ERR_NULL;
    if (g.n_tokens < 0 || g.n_tokens > kLatentMaxTokens / 4 || g.heads <= 0 || g.heads > kLatentMaxHeads) return VIB3_ERR_COUNT;
    if (dtype != L_F16 && dtype != L_BF16) return VIB3_ERR_UNSUPPORTED;
    if (g.dim < 16 || g.dim > 256 || g.dim % 16) return VIB3_ERR_UNSUPPORTED;
    // rows of the result may not overlap; rows of the inputs may repeat (a stride of zero broadcasts)
    if (g.a_token < 0 || g.a_head < 0 || g.w_head < 0 || (g.heads > 1 && g.out_head < out_width) || (g.n_tokens > 1 && g.out_token < out_width))
        return VIB3_ERR_SHAPE;
    if (off16(g.a) || off16(g.w) || off16(g.out) || g.a_token % 8 || g.a_head % 8 || g.w_head % 8 || g.out_token % 8 || g.out_head % 8)
        return VIB3_ERR_ALIGN;
    return VIB3_OK;
}

extern "C" int vib3_launch_latent_query(const void* q, long long q_token_stride, long long q_head_stride, const void* w_uk,
                                        long long w_head_stride, const int* positions, const double* inv_freq, float rope_scale, int pairs,
                                        void* out, long long out_token_stride, long long out_head_stride, int n_tokens, int heads, int nope,
                                        int dtype, int* status, void* stream) {
    HeadArgs g{q, q_token_stride, q_head_stride, w_uk, w_head_stride, out, out_token_stride, out_head_stride, n_tokens, heads, nope,
               positions, inv_freq, rope_scale, pairs, status};
    if ((n_tokens != 0 && !positions) || !inv_freq) return VIB3_ERR_NULL;
    const int e = check_heads(g, dtype, kLatentRow);
    if (e) return e;
    if (n_tokens == 0) return VIB3_OK;
    return dtype == L_F16 ? launch_heads<__half, true>(g, dtype, (cudaStream_t)stream) : launch_heads<__nv_bfloat16, true>(g, dtype, (cudaStream_t)stream);
}

extern "C" int vib3_launch_latent_value(const void* o, long long o_token_stride, long long o_head_stride, const void* w_uv,
                                        long long w_head_stride, void* out, long long out_token_stride, long long out_head_stride,
                                        int n_tokens, int heads, int value, int dtype, int* status, void* stream) {
    HeadArgs g{o, o_token_stride, o_head_stride, w_uv, w_head_stride, out, out_token_stride, out_head_stride, n_tokens, heads, value,
               nullptr, nullptr, 1.f, 0, status};
    const int e = check_heads(g, dtype, value);
    if (e) return e;
    if (n_tokens == 0) return VIB3_OK;
    return dtype == L_F16 ? launch_heads<__half, false>(g, dtype, (cudaStream_t)stream) : launch_heads<__nv_bfloat16, false>(g, dtype, (cudaStream_t)stream);
}
