// The steps of a latent-attention layer around the attention itself:
//   vib3_launch_latent_append_paged   normalise, rotate and store a step's rows into the paged cache
//   vib3_launch_latent_query          per head q_nope . W_uk and the rotation of q_rope
//   vib3_launch_latent_value          per head o . W_uv^T
// The reference has a scalar kernel for each (vib3_mla_kv_cache_append_kernel, vib3_mla_q_absorb_rope_kernel,
// vib3_mla_v_reconstruct, cuda/src/kernels.cu:1709, :1679, :1624), for one token and a flat cache.
#include "latent_common.cuh"

namespace vib3 {

// ── append ───────────────────────────────────────────────────────────────────────────────────
// row[0:512] = x / sqrt(mean(x^2) + eps) * w, row[512:576] = rotated x, rounded once.  One warp per token: the row stays in
// registers between the sum of squares and the scaling, so a token is read once and written once.  Bound by the launch for a
// decode step, by HBM for a prompt.
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
// C[t, n] = sum_k A[t, k] B(k, n) for one head, fp32 accumulation on the warp-level tensor instructions.  These products are
// bound by their bytes, not by their arithmetic: with one token the head matrices are read for two flops per value, with 512 a
// query's result rows are most of the traffic.
constexpr int kChunkK = 64;   // columns of K per pipeline stage: 128-byte rows

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes global -> shared, zeros where !valid (the address is then not read)
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldm4(uint32_t a, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldm2(uint32_t a, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t a, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16(float* d, const uint32_t* a, const uint32_t* b) {
    if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// One BM x BN tile.  NK: B is stored [n][k] (k contiguous), else [k][n].  Tiles lie in shared memory as rows of 128 bytes (B as
// [k][n]: 2 BN bytes) whose 16-byte pieces are permuted by the row number, so that the eight rows of a matrix fragment come
// from different banks.  Rows and columns outside the matrix are zeros, so their values in memory do not matter.
template <typename T, bool NK, int BM_, int BN_, int WARPS_M, int WARPS_N, int STAGES>
struct HeadTile {
    static constexpr int BM = BM_, BN = BN_;
    static constexpr int kThreads = WARPS_M * WARPS_N * 32;
    static constexpr int WM = BM / WARPS_M, WN = BN / WARPS_N, MF = WM / 16, NF = WN / 8;
    static constexpr int kABytes = BM * kChunkK * 2, kBBytes = BN * kChunkK * 2;
    static constexpr int kOutStride = BN + 8;
    static constexpr size_t kPipe = (size_t)STAGES * (kABytes + kBBytes), kOut = (size_t)BM * kOutStride * 2;
    static constexpr size_t kSmem = kPipe > kOut ? kPipe : kOut;
    static_assert(MF >= 1 && (NF == 1 || NF % 2 == 0) && (NK || NF % 2 == 0), "fragments");
    static_assert(NK || BN >= 64, "a row of B holds the eight permuted pieces");

    // A: rows t0.. of T rows, a_stride elements apart; B: n0.. of N; the result goes to c (row stride c_stride).
    static __device__ void run(unsigned char* smem, const T* A, long long a_stride, int t0, int n_tokens, const T* B, int b_stride, int n0,
                               int N, int K, T* C, long long c_stride) {
        const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
        const int wm = warp / WARPS_N, wn = warp % WARPS_N;
        const uint32_t base = smem_addr(smem);
        const int nk = (K + kChunkK - 1) / kChunkK;
        auto load = [&](int kc) {
            const uint32_t sa = base + (kc % STAGES) * (kABytes + kBBytes), sb = sa + kABytes;
            const int k0 = kc * kChunkK;
#pragma unroll
            for (int i = tid; i < BM * 8; i += kThreads) {
                const int r = i >> 3, c = i & 7;
                const bool ok = t0 + r < n_tokens && k0 + c * 8 < K;
                cp16(sa + r * 128 + ((c ^ (r & 7)) << 4), ok ? A + (long long)(t0 + r) * a_stride + k0 + c * 8 : A, ok);
            }
            if constexpr (NK) {
#pragma unroll
                for (int i = tid; i < BN * 8; i += kThreads) {
                    const int r = i >> 3, c = i & 7;
                    const bool ok = n0 + r < N && k0 + c * 8 < K;
                    cp16(sb + r * 128 + ((c ^ (r & 7)) << 4), ok ? B + (long long)(n0 + r) * b_stride + k0 + c * 8 : B, ok);
                }
            } else {
                constexpr int P = BN / 8;   // 16-byte pieces of a row
#pragma unroll
                for (int i = tid; i < kChunkK * P; i += kThreads) {
                    const int r = i / P, c = i % P;
                    const bool ok = k0 + r < K && n0 + c * 8 < N;
                    cp16(sb + r * (BN * 2) + ((c ^ (r & 7)) << 4), ok ? B + (long long)(k0 + r) * b_stride + n0 + c * 8 : B, ok);
                }
            }
        };
        float acc[MF][NF][4];
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int j = 0; j < NF; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.f;
#pragma unroll
        for (int s = 0; s < STAGES; ++s) {
            if (s < nk) load(s);
            cp_commit();
        }
        for (int kc = 0; kc < nk; ++kc) {
            cp_wait<STAGES - 1>();
            __syncthreads();
            const uint32_t sa = base + (kc % STAGES) * (kABytes + kBBytes), sb = sa + kABytes;
#pragma unroll
            for (int ks = 0; ks < kChunkK / 16; ++ks) {
                uint32_t af[MF][4], bf[NF][2];
#pragma unroll
                for (int i = 0; i < MF; ++i) {
                    const int r = wm * WM + i * 16 + (lane & 15), c = ks * 2 + (lane >> 4);
                    ldm4(sa + r * 128 + ((c ^ (r & 7)) << 4), af[i]);
                }
                if constexpr (NF == 1) {
                    const int r = wn * WN + (lane & 7), c = ks * 2 + ((lane >> 3) & 1);
                    ldm2(sb + r * 128 + ((c ^ (r & 7)) << 4), bf[0]);
                } else {
#pragma unroll
                    for (int j = 0; j < NF; j += 2) {
                        if constexpr (NK) {
                            const int r = wn * WN + j * 8 + (lane & 7) + ((lane >> 4) << 3), c = ks * 2 + ((lane >> 3) & 1);
                            ldm4(sb + r * 128 + ((c ^ (r & 7)) << 4), bf[j]);
                        } else {
                            const int r = ks * 16 + (lane & 15), c = (wn * WN + j * 8) / 8 + (lane >> 4);
                            ldm4t(sb + r * (BN * 2) + ((c ^ (r & 7)) << 4), bf[j]);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < MF; ++i)
#pragma unroll
                    for (int j = 0; j < NF; ++j) mma16<T>(acc[i][j], af[i], bf[j]);
            }
            __syncthreads();
            if (kc + STAGES < nk) load(kc + STAGES);
            cp_commit();
        }
        // the tile through shared memory, so that a row leaves in 16-byte pieces
        cp_wait<0>();
        __syncthreads();
        T* so = reinterpret_cast<T*>(smem);
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int j = 0; j < NF; ++j) {
                const int r = wm * WM + i * 16 + (lane >> 2), c = wn * WN + j * 8 + (lane & 3) * 2;
                *reinterpret_cast<uint32_t*>(so + r * kOutStride + c) = pack2<T>(acc[i][j][0], acc[i][j][1]);
                *reinterpret_cast<uint32_t*>(so + (r + 8) * kOutStride + c) = pack2<T>(acc[i][j][2], acc[i][j][3]);
            }
        __syncthreads();
        for (int i = tid; i < BM * (BN / 8); i += kThreads) {
            const int r = i / (BN / 8), c = (i % (BN / 8)) * 8;
            if (t0 + r < n_tokens && n0 + c < N)
                *reinterpret_cast<uint4*>(C + (long long)(t0 + r) * c_stride + n0 + c) = *reinterpret_cast<const uint4*>(so + r * kOutStride + c);
        }
    }
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
    int product_blocks;          // blocks of the product; the others rotate
};

// blockIdx.x = (tile of tokens * heads + head) * column blocks + column block.
template <typename T, class Tile>
__global__ void __launch_bounds__(Tile::kThreads) latent_value_kernel(HeadArgs g) {
    extern __shared__ __align__(128) unsigned char smem[];
    pdl_enter();
    const int nb = (g.dim + Tile::BN - 1) / Tile::BN;
    const int n = blockIdx.x % nb, h = blockIdx.x / nb % g.heads, tt = blockIdx.x / nb / g.heads;
    Tile::run(smem, (const T*)g.a + h * g.a_head, g.a_token, tt * Tile::BM, g.n_tokens, (const T*)g.w + h * g.w_head, kRank, n * Tile::BN,
              g.dim, kRank, (T*)g.out + h * g.out_head, g.out_token);
}

constexpr int kRotateHeads = 16;   // heads that share one evaluation of a token's angles

template <typename T, class Tile>
__global__ void __launch_bounds__(Tile::kThreads) latent_query_kernel(HeadArgs g) {
    extern __shared__ __align__(128) unsigned char smem[];
    pdl_enter();
    if ((int)blockIdx.x < g.product_blocks) {
        constexpr int nb = kRank / Tile::BN;
        const int n = blockIdx.x % nb, h = blockIdx.x / nb % g.heads, tt = blockIdx.x / nb / g.heads;
        Tile::run(smem, (const T*)g.a + h * g.a_head, g.a_token, tt * Tile::BM, g.n_tokens, (const T*)g.w + h * g.w_head, kRank,
                  n * Tile::BN, kRank, g.dim, (T*)g.out + h * g.out_head, g.out_token);
        return;
    }
    // the rotation: a warp turns the 64 position values of up to 16 heads of one token
    const int lane = threadIdx.x & 31;
    const int groups = (g.heads + kRotateHeads - 1) / kRotateHeads;
    const int item = (blockIdx.x - g.product_blocks) * (Tile::kThreads / 32) + (threadIdx.x >> 5);
    if (item >= g.n_tokens * groups) return;
    const int t = item / groups, h0 = item % groups * kRotateHeads, hn = min(kRotateHeads, g.heads - h0);
    const T* q = (const T*)g.a + t * g.a_token + h0 * g.a_head + g.dim;
    T* o = (T*)g.out + t * g.out_token + h0 * g.out_head + kRank;
    const int i0 = g.pairs ? 2 * lane : lane, i1 = g.pairs ? 2 * lane + 1 : lane + 32;
    float c, s;
    rope_angle(g.positions[t], g.inv_freq[lane], g.rope_scale, c, s);
#pragma unroll 8
    for (int h = 0; h < hn; ++h) {
        const T* x = q + h * g.a_head;
        T* y = o + h * g.out_head;
        const float a = as_float(x[i0]), b = as_float(x[i1]);
        y[i0] = from_float<T>(a * c - b * s);
        y[i1] = from_float<T>(b * c + a * s);
    }
}

namespace {

template <class K>
int allow_smem(K kernel, size_t bytes) {
    if (bytes <= 48 * 1024) return 0;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != cudaSuccess) (void)cudaGetLastError();
    return (int)e;
}

int ceil_div(int a, int b) { return (a + b - 1) / b; }

template <typename T, class Tile>
int launch_value(const HeadArgs& g, cudaStream_t st) {
    const int e = allow_smem(latent_value_kernel<T, Tile>, Tile::kSmem);
    if (e) return e;
    const dim3 grid((unsigned)(ceil_div(g.dim, Tile::BN) * g.heads * ceil_div(g.n_tokens, Tile::BM)));
    return launch_latent(latent_value_kernel<T, Tile>, grid, Tile::kThreads, Tile::kSmem, st, g);
}

template <typename T, class Tile>
int launch_query(HeadArgs g, cudaStream_t st) {
    const int e = allow_smem(latent_query_kernel<T, Tile>, Tile::kSmem);
    if (e) return e;
    g.product_blocks = kRank / Tile::BN * g.heads * ceil_div(g.n_tokens, Tile::BM);
    const int rotate = ceil_div(g.n_tokens * ceil_div(g.heads, kRotateHeads), Tile::kThreads / 32);
    return launch_latent(latent_query_kernel<T, Tile>, dim3((unsigned)(g.product_blocks + rotate)), Tile::kThreads, Tile::kSmem, st, g);
}

template <typename T>
int value_of(const HeadArgs& g, cudaStream_t st) {
    if (g.n_tokens <= 16) return launch_value<T, HeadTile<T, true, 16, 32, 1, 4, 8>>(g, st);
    return launch_value<T, HeadTile<T, true, 64, 64, 2, 4, 4>>(g, st);
}

template <typename T>
int query_of(const HeadArgs& g, cudaStream_t st) {
    if (g.n_tokens <= 16) return launch_query<T, HeadTile<T, false, 16, 128, 1, 4, 2>>(g, st);
    return launch_query<T, HeadTile<T, false, 64, 128, 2, 4, 2>>(g, st);
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
    if (!kv || !positions || !slots || !inv_freq || !cache) return VIB3_ERR_NULL;
    if (n_tokens < 0 || n_tokens > kLatentMaxTokens || num_pages <= 0 || page_size <= 0) return VIB3_ERR_COUNT;
    if (kv_dtype < L_F32 || kv_dtype > L_BF16 || (cache_dtype != L_F16 && cache_dtype != L_BF16)) return VIB3_ERR_UNSUPPORTED;
    if (row_stride < kLatentRow || page_stride < 0 || (n_tokens > 1 && kv_stride < kLatentRow)) return VIB3_ERR_SHAPE;
    const int per16 = kv_dtype == L_F32 ? 4 : 8;
    if (off16(kv) || kv_stride % per16 || off16(norm_weight_or_null) || off16(cache) || page_stride % 8 || row_stride % 8) return VIB3_ERR_ALIGN;
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

static int check_heads(const HeadArgs& g, int dtype, int in_width, int out_width) {
    if (!g.a || !g.w || !g.out) return VIB3_ERR_NULL;
    if (g.n_tokens < 0 || g.n_tokens > kLatentMaxTokens / 4 || g.heads <= 0 || g.heads > kLatentMaxHeads) return VIB3_ERR_COUNT;
    if (dtype != L_F16 && dtype != L_BF16) return VIB3_ERR_UNSUPPORTED;
    if (g.dim < 16 || g.dim > 256 || g.dim % 16) return VIB3_ERR_UNSUPPORTED;
    // rows of the result may not overlap; rows of the inputs may repeat (a stride of zero broadcasts)
    if (g.a_token < 0 || g.a_head < 0 || g.w_head < 0 || (g.heads > 1 && g.out_head < out_width) || (g.n_tokens > 1 && g.out_token < out_width))
        return VIB3_ERR_SHAPE;
    (void)in_width;
    if (off16(g.a) || off16(g.w) || off16(g.out) || g.a_token % 8 || g.a_head % 8 || g.w_head % 8 || g.out_token % 8 || g.out_head % 8)
        return VIB3_ERR_ALIGN;
    return VIB3_OK;
}

extern "C" int vib3_launch_latent_query(const void* q, long long q_token_stride, long long q_head_stride, const void* w_uk,
                                        long long w_head_stride, const int* positions, const double* inv_freq, float rope_scale, int pairs,
                                        void* out, long long out_token_stride, long long out_head_stride, int n_tokens, int heads, int nope,
                                        int dtype, void* stream) {
    HeadArgs g{q, q_token_stride, q_head_stride, w_uk, w_head_stride, out, out_token_stride, out_head_stride, n_tokens, heads, nope,
               positions, inv_freq, rope_scale, pairs, 0};
    if (!positions || !inv_freq) return VIB3_ERR_NULL;
    const int e = check_heads(g, dtype, nope + kRope, kLatentRow);
    if (e) return e;
    if (n_tokens == 0) return VIB3_OK;
    return dtype == L_F16 ? query_of<__half>(g, (cudaStream_t)stream) : query_of<__nv_bfloat16>(g, (cudaStream_t)stream);
}

extern "C" int vib3_launch_latent_value(const void* o, long long o_token_stride, long long o_head_stride, const void* w_uv,
                                        long long w_head_stride, void* out, long long out_token_stride, long long out_head_stride,
                                        int n_tokens, int heads, int value, int dtype, void* stream) {
    HeadArgs g{o, o_token_stride, o_head_stride, w_uv, w_head_stride, out, out_token_stride, out_head_stride, n_tokens, heads, value,
               nullptr, nullptr, 1.f, 0, 0};
    const int e = check_heads(g, dtype, kRank, value);
    if (e) return e;
    if (n_tokens == 0) return VIB3_OK;
    return dtype == L_F16 ? value_of<__half>(g, (cudaStream_t)stream) : value_of<__nv_bfloat16>(g, (cudaStream_t)stream);
}
