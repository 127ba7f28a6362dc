// Latent attention in the absorbed form over a paged cache.
//
// Row r of sequence b is (token j, head h) of its q_len newest tokens; token j stands at position p = len - q_len + j and sees
// the keys 0 .. p.  With q and c_k rows of 576 values, of which the first 512 are the value too:
//   s_k = scale * q . c_k,   lse = log sum_{k <= p} exp(s_k),   o = sum_{k <= p} exp(s_k - lse) c_k[0:512]
// A row that sees nothing gives o = 0 and lse = -inf.
#include "latent_common.cuh"

namespace vib3 {

struct AttentionArgs {
    const void* q;
    long long q_token, q_head;             // strides in elements
    const void* cache;
    long long num_pages;
    int page_size;
    long long page_stride, row_stride;     // elements
    const int* page_table;
    int table_stride, max_pages;
    const int* seq_lens;
    int batch, q_len, heads;
    float scale;
    void* out;
    long long out_token, out_head;
    float* lse;
    int* status;
};

constexpr int kSimpleKeys = 16, kSimpleWarps = 8;

template <typename T>
__global__ void __launch_bounds__(kSimpleWarps * 32) latent_attention_kernel(AttentionArgs a) {
    __shared__ __align__(16) T keys[kSimpleKeys][kLatentRow];
    __shared__ int valid[kSimpleKeys];
    pdl_enter();
    const int t = blockIdx.x, b = t / a.q_len, j = t % a.q_len;
    const int lane = threadIdx.x & 31, h = blockIdx.y * kSimpleWarps + (threadIdx.x >> 5);
    const int seen = max(a.seq_lens[b] - a.q_len + j + 1, 0);
    float q[18], o[16], m = -INFINITY, l = 0.f;
    const T* qp = (const T*)a.q + t * a.q_token + min(h, a.heads - 1) * a.q_head;
#pragma unroll
    for (int i = 0; i < 18; ++i) q[i] = as_float(qp[lane + 32 * i]) * a.scale;
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = 0.f;
    for (int k0 = 0; k0 < seen; k0 += kSimpleKeys) {
        const int n = min(kSimpleKeys, seen - k0);
        __syncthreads();
        for (int i = threadIdx.x; i < n * (kLatentRow / 8); i += blockDim.x) {
            const int r = i / (kLatentRow / 8), c = i % (kLatentRow / 8), k = k0 + r, pi = k / a.page_size;
            const int page = pi < a.max_pages ? a.page_table[(long long)b * a.table_stride + pi] : -1;
            const bool ok = page >= 0 && page < a.num_pages;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (ok) v = *reinterpret_cast<const uint4*>((const T*)a.cache + page * a.page_stride + (k % a.page_size) * a.row_stride + c * 8);
            *reinterpret_cast<uint4*>(&keys[r][c * 8]) = v;
            if (c == 0) {
                valid[r] = ok;
                if (!ok && a.status) atomicOr(a.status, kStatusBadPage);
            }
        }
        __syncthreads();
        for (int r = 0; r < n; ++r) {
            if (!valid[r]) continue;
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < 18; ++i) s = fmaf(q[i], as_float(keys[r][lane + 32 * i]), s);
#pragma unroll
            for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
            const float mn = fmaxf(m, s), f = m == -INFINITY ? 0.f : expf(m - mn), p = mn == -INFINITY ? 0.f : expf(s - mn);
            l = l * f + p;
            m = mn;
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = fmaf(o[i], f, p * as_float(keys[r][lane + 32 * i]));
        }
    }
    if (h >= a.heads) return;
    const float inv = l > 0.f ? 1.f / l : 0.f;
    T* out = (T*)a.out + t * a.out_token + h * a.out_head;
#pragma unroll
    for (int i = 0; i < 16; ++i) out[lane + 32 * i] = from_float<T>(o[i] * inv);
    if (lane == 0 && a.lse) a.lse[(long long)t * a.heads + h] = l > 0.f ? m + logf(l) : -INFINITY;
}

}  // namespace vib3

using namespace vib3;

extern "C" size_t vib3_latent_attention_workspace_bytes(void) { return 48u << 20; }

extern "C" int vib3_launch_latent_attention_paged(const void* q, long long q_token_stride, long long q_head_stride, const void* cache,
                                                  long long num_pages, int page_size, long long page_stride, long long row_stride,
                                                  const int* page_table, int table_stride, int max_pages_per_seq, const int* seq_lens,
                                                  int batch, int q_len, int heads, float scale, int dtype, void* out,
                                                  long long out_token_stride, long long out_head_stride, float* lse_or_null,
                                                  void* workspace, size_t workspace_bytes, int* status, void* stream) {
    if (!q || !cache || !page_table || !seq_lens || !out || !workspace) return VIB3_ERR_NULL;
    if (dtype != L_F16 && dtype != L_BF16) return VIB3_ERR_UNSUPPORTED;
    if (page_size % 8) return VIB3_ERR_UNSUPPORTED;
    if (batch < 0 || q_len < 0 || heads <= 0 || heads > kLatentMaxHeads || num_pages <= 0 || num_pages > 0x7fffffff || page_size <= 0 ||
        page_size > (1 << 20) || max_pages_per_seq <= 0 || (long long)max_pages_per_seq * page_size > 0x7fffffff ||
        (long long)batch * q_len > (1 << 20))
        return VIB3_ERR_COUNT;
    if (row_stride < kLatentRow || page_stride < row_stride * (page_size - 1) + kLatentRow || q_token_stride < 0 || q_head_stride < 0 ||
        (batch > 1 && table_stride < max_pages_per_seq) || (heads > 1 && out_head_stride < kRank) ||
        ((long long)batch * q_len > 1 && out_token_stride < kRank))
        return VIB3_ERR_SHAPE;
    if (((uintptr_t)q & 15) || ((uintptr_t)cache & 15) || ((uintptr_t)out & 15) || ((uintptr_t)workspace & 15) || q_token_stride % 8 ||
        q_head_stride % 8 || page_stride % 8 || row_stride % 8 || out_token_stride % 8 || out_head_stride % 8)
        return VIB3_ERR_ALIGN;
    if (workspace_bytes < vib3_latent_attention_workspace_bytes()) return VIB3_ERR_CAPACITY;
    if (batch == 0 || q_len == 0) return VIB3_OK;
    AttentionArgs a{q, q_token_stride, q_head_stride, cache, num_pages, page_size, page_stride, row_stride, page_table, table_stride,
                    max_pages_per_seq, seq_lens, batch, q_len, heads, scale, out, out_token_stride, out_head_stride, lse_or_null, status};
    const dim3 grid((unsigned)(batch * q_len), (unsigned)((heads + kSimpleWarps - 1) / kSimpleWarps));
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == L_F16) return launch_latent(latent_attention_kernel<__half>, grid, kSimpleWarps * 32, 0, st, a);
    return launch_latent(latent_attention_kernel<__nv_bfloat16>, grid, kSimpleWarps * 32, 0, st, a);
}
