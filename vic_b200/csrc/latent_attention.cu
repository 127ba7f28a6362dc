// Latent attention in the absorbed form over a paged cache.
//
// Row r of sequence b is (token j, head h) of its q_len newest tokens, r = j * heads + h; token j stands at position p = len -
// q_len + j and sees the keys 0 .. p.  With q and c_k rows of 576 values, of which the first 512 are the value too:
//   s_k = scale * q . c_k,   lse = log sum_{k <= p} exp(s_k),   o = sum_{k <= p} exp(s_k - lse) c_k[0:512]
// A row that sees nothing gives o = 0 and lse = -inf.  One pass over the keys in tiles of 64: with the running reference m,
//   p_k = exp(s_k - m),  l += sum p_k,  O += p_k c_k;   when m moves to m', l and O are multiplied by exp(m - m').
//
// What bounds it: a cache row of 1152 bytes serves 2 (576 + 512) flops per row r, 121 flops per byte with 64 heads, half of
// what the card does per byte; so HBM, as long as the tensor pipe keeps up.  Warp-level MMAs (about a third of the tcgen05
// rate) do not.  Hence per tile of 64 keys and block of 64 rows, one CTA per SM:
//   S [64 rows x 64 keys]  = Q . C^T      tcgen05, M = 64, K = 576; Q stays in shared memory for the whole sequence
//   P = exp(S - m)                        four warps, from tensor memory to shared memory as 16-bit values
//   O^T [512 x 64 rows]   += C^T . P^T    tcgen05, four products with M = 128 values and N = 64 rows
// The tile of C that TMA brought once is operand of both products: K-major (its 576 values contiguous) in the first, and in the
// second, through another descriptor of the same bytes, MN-major.  With the accumulator transposed its 256 columns fill all 128
// lanes of tensor memory, so it stays there for the whole sequence, and the number of rows is the N of the MMA.  Q (72 KB), two
// tiles (144 KB) and P (8 KB) are all of shared memory; the tiles are handed over in five pieces of 128 (64) values, so that a
// piece is refilled as soon as its product has read it.
#include <cuda.h>

#include "latent_common.cuh"

namespace vib3 {

int sm_count();

constexpr int kTileKeys = 64, kTileRows = 64;
constexpr int kChunkBytes = 64 * 128;                     // 64 rows of 64 values, 128-byte swizzle
constexpr int kChunks = kLatentRow / 64;                  // 9: eight of the latent, one of position values
constexpr int kTileBytes = kChunks * kChunkBytes;
constexpr int kGroups = 5;                                // pieces of a tile: chunk pairs 0..3, the position chunk
constexpr int kQOff = 0, kKvOff = kTileBytes, kPOff = 3 * kTileBytes, kMiscOff = kPOff + kChunkBytes;
constexpr int kAttThreads = 256;                          // copies, MMAs, two warps for Q, four for the softmax and the results
constexpr int kSoftmaxThreads = 128;
constexpr int kTmemCols = 512, kSCol = 256;               // O^T: 4 x 64 columns, S: 2 x 64
// The reference m of a row follows its maximum only when that has grown by more than 2^8: exp(s - m) then stays below 256, the
// 16-bit weights keep their relative precision, and the accumulator is rescaled a few times per sequence instead of per tile.
constexpr float kLazy = 8.0f;
constexpr int kMaxGrid = 160;                             // CTAs that the workspace has room for
constexpr size_t kPartFloats = (size_t)kTileRows * kRank;

struct AttentionArgs {
    const void* q;
    long long q_token, q_head;             // strides in elements
    int page_size, box_rows;
    int num_pages;
    const int* page_table;
    int table_stride, max_pages;
    const int* seq_lens;
    int batch, q_len, heads;
    float scale_log2;                      // scale * log2(e)
    void* out;
    long long out_token, out_head;
    float* lse;
    int* status;
    int lanes, blocks_per_lane;            // see Plan
    int min_tiles;
    // workspace: what CTA c owes to a sequence that other CTAs share, two slots per CTA
    int4* owner;                           // [grid] sequence, row block, parts (0: none)
    float2* part_ml;                       // [2 grid][64] reference (log2) and sum
    float* part_o;                         // [2 grid][64][512], not yet divided by the sum
};

// The split.  A sequence has row blocks of 64 rows, a row block as many tiles as its last row sees.  Few row blocks (lanes =
// their number): CTA = share * lanes + row block, so that the CTAs of a share read the same tiles at the same time and the cache
// comes from HBM once.  Many: one lane, and a sequence's row blocks follow one another.  Within a lane the tiles of all sequences form one line that
// is cut into equal shares whatever the lengths are; a sequence that a cut divides leaves parts that a second launch adds up.
struct Plan {
    long long begin, end, total;           // this CTA's tiles on the line
    long long prefix;                      // of the first item
    int item, lane, share, shares;
};

struct Piece {
    int b, rb, seen, tiles;                // item: sequence, row block, keys of its last row, tiles
    int t0, t1;                            // this CTA's tiles of it
    long long prefix;
};

__device__ __forceinline__ int item_count(const AttentionArgs& a) { return a.batch * a.blocks_per_lane; }

__device__ __forceinline__ void item_of(const AttentionArgs& a, int lane, int item, Piece& p) {
    p.b = a.blocks_per_lane == 1 ? item : item / a.blocks_per_lane;
    p.rb = lane * a.blocks_per_lane + (item - p.b * a.blocks_per_lane);
    const int last_row = min(a.q_len * a.heads, (p.rb + 1) * kTileRows) - 1;
    const int len = max(__ldg(a.seq_lens + p.b), 0);
    p.seen = min(max(len - a.q_len + last_row / a.heads + 1, 0), a.max_pages * a.page_size);
    p.tiles = (p.seen + kTileKeys - 1) / kTileKeys;
}

// The pieces of this CTA in order.  Items without tiles belong to the CTA whose share they stand in (t0 == t1).
struct Walk {
    const AttentionArgs& a;
    const Plan& plan;
    int item, items;
    long long prefix;
    __device__ __forceinline__ Walk(const AttentionArgs& a_, const Plan& p_) : a(a_), plan(p_), item(p_.item), items(item_count(a_)), prefix(p_.prefix) {}
    __device__ __forceinline__ bool next(Piece& p, bool with_empty) {
        const bool last = plan.share == plan.shares - 1;
        while (item < items && (prefix < plan.end || last)) {
            item_of(a, plan.lane, item, p);
            p.prefix = prefix;
            ++item;
            prefix += p.tiles;
            if (p.tiles == 0) {
                p.t0 = p.t1 = 0;
                if (with_empty) return true;
                continue;
            }
            p.t0 = (int)max(plan.begin - p.prefix, 0ll);
            p.t1 = (int)min(plan.end - p.prefix, (long long)p.tiles);
            if (p.t1 > p.t0) return true;
        }
        return false;
    }
};

struct AttShared {
    uint64_t kv_full[2][kGroups], kv_empty[2][kGroups];
    uint64_t s_full[2], p_full, pv_done, q_full, q_empty, drain;
    unsigned long long mask[2];            // keys of the tile that count
    alignas(16) float factor[2][kTileRows];
    alignas(16) float inv[kTileRows];
    Plan plan;
    long long warp_sum[kAttThreads / 32];
    uint32_t tmem;
};
static_assert(kMiscOff + sizeof(AttShared) <= 227 * 1024, "shared memory of a CTA");
constexpr int kAttSmem = kMiscOff + (int)sizeof(AttShared);

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint64_t* bar, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t* bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Waits for the phase with this parity; gives up, with false, after about four seconds (a try comes back after some 4 us).
__device__ __forceinline__ bool bar_wait(uint64_t* bar, unsigned parity) {
    const uint32_t addr = smem_u32(bar);
    uint32_t ok = 0;
    for (unsigned it = 0; !ok && it < (1u << 20); ++it)
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(addr), "r"(parity) : "memory");
    return ok != 0;
}
// The same for a whole warp, whose lanes have to agree (they meet again in warp-wide instructions).
__device__ __forceinline__ bool bar_wait_warp(uint64_t* bar, unsigned parity) { return __all_sync(0xffffffffu, bar_wait(bar, parity)); }
// One lane of the warp, the same one every time: behind elect.sync MMAs and tensor copies issue back to back.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Named barrier of the softmax warps; the second form tells whether any of them says so.
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kSoftmaxThreads) : "memory"); }
__device__ __forceinline__ bool softmax_any(bool v) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"((uint32_t)v), "n"(kSoftmaxThreads) : "memory");
    return r != 0;
}

// Shared-memory operands with 128-byte swizzle.  K-major: rows of 128 bytes, eight of them 1024 bytes.  MN-major: 64 values
// contiguous per key, eight keys 1024 bytes, the next 64 values a chunk further.
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)(kChunkBytes >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}
template <typename T> constexpr uint32_t kFormat = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
template <typename T> constexpr uint32_t kIdescS = (1u << 4) | (kFormat<T> << 7) | (kFormat<T> << 10) | (64u / 8 << 17) | (64u / 16 << 24);
template <typename T> constexpr uint32_t kIdescO = (1u << 4) | (kFormat<T> << 7) | (kFormat<T> << 10) | (1u << 15) | (64u / 8 << 17) | (128u / 16 << 24);

__device__ __forceinline__ void tmem_ld_16x64(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr) : "memory");
}

__device__ __forceinline__ void tmem_ld_32x32(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr) : "memory");
}

__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}

// This CTA's place on its lane's line of tiles.  All threads.
__device__ __forceinline__ void make_plan(const AttentionArgs& a, AttShared& sh) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row_lane = blockIdx.x % a.lanes, share = blockIdx.x / a.lanes, items = item_count(a);
    Piece p;
    auto block_sum = [&](long long v) {
#pragma unroll
        for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
        __syncthreads();
        if (lane == 0) sh.warp_sum[warp] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int w = 0; w < kAttThreads / 32; ++w) v += sh.warp_sum[w];
        return v;
    };
    long long mine = 0;
    for (int i = tid; i < items; i += kAttThreads) {
        item_of(a, row_lane, i, p);
        mine += p.tiles;
    }
    const long long total = block_sum(mine);
    const int most = gridDim.x / a.lanes;
    const int shares = (int)max(1ll, min((long long)most, (total + a.min_tiles - 1) / a.min_tiles));
    const long long begin = share < shares ? total * share / shares : total, end = share < shares ? total * (share + 1) / shares : total;
    if (tid == 0) {
        sh.plan.begin = begin; sh.plan.end = end; sh.plan.total = total;
        sh.plan.item = items; sh.plan.prefix = total; sh.plan.lane = row_lane; sh.plan.share = share; sh.plan.shares = shares;
    }
    if (share >= shares) {
        __syncthreads();
        return;
    }
    // the first item that begins at `begin` or reaches beyond it
    long long base = 0;
    for (int i0 = 0; i0 < items; i0 += kAttThreads) {
        const int i = i0 + tid;
        long long tiles = 0;
        if (i < items) {
            item_of(a, row_lane, i, p);
            tiles = p.tiles;
        }
        long long incl = tiles;
#pragma unroll
        for (int m = 1; m < 32; m <<= 1) {
            const long long o = __shfl_up_sync(0xffffffffu, incl, m);
            if (lane >= m) incl += o;
        }
        __syncthreads();
        if (lane == 31) sh.warp_sum[warp] = incl;
        __syncthreads();
        long long before = base;
        for (int w = 0; w < warp; ++w) before += sh.warp_sum[w];
        const long long pre = before + incl - tiles;
        const bool mineIs = i < items && (pre == begin || pre + tiles > begin);
        // (one thread: the item before it does not qualify)
        const unsigned hits = __ballot_sync(0xffffffffu, mineIs);
        bool first = mineIs && (hits & ((1u << lane) - 1)) == 0;
        if (first && lane == 0 && i > 0) {   // the previous item is another warp's (or chunk's)
            Piece prev;
            item_of(a, row_lane, i - 1, prev);
            const long long ppre = pre - prev.tiles;
            first = !(ppre == begin || pre > begin);
        }
        if (first) {
            sh.plan.item = i;
            sh.plan.prefix = pre;
        }
        for (int w = 0; w < kAttThreads / 32; ++w) base += sh.warp_sum[w];
        if (base > begin) break;
    }
    __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kAttThreads, 1) latent_attention_kernel(const __grid_constant__ CUtensorMap map, const AttentionArgs a) {
    extern __shared__ __align__(1024) unsigned char smem[];
    AttShared& sh = *reinterpret_cast<AttShared*>(smem + kMiscOff);
    const uint32_t base = smem_u32(smem);
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    if (tid == 0) {
        for (int s = 0; s < 2; ++s) {
            for (int g = 0; g < kGroups; ++g) {
                bar_init(&sh.kv_full[s][g], 1);
                bar_init(&sh.kv_empty[s][g], 1);
            }
            bar_init(&sh.s_full[s], 1);
        }
        bar_init(&sh.p_full, kSoftmaxThreads);
        bar_init(&sh.pv_done, 1);
        bar_init(&sh.q_full, 64);
        bar_init(&sh.q_empty, 1);
        bar_init(&sh.drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "n"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == 0 && elect_one()) asm volatile("prefetch.tensormap [%0];" ::"l"(&map) : "memory");
    pdl_enter();
    make_plan(a, sh);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const Plan& plan = sh.plan;
    const int rows_all = a.q_len * a.heads;
    Walk walk(a, plan);
    Piece p;
    bool ok = (base & 1023) == 0;   // the swizzle is a function of the address

    if (warp == 0) {
        // ── copies: the tiles of C, in boxes of box_rows rows that lie in one page ──
        const int R = a.box_rows, nb = kTileKeys / R, per_load = 32 / nb;
        int it = 0, issued = kGroups;   // pieces of the newest tile that were requested
        while (ok && walk.next(p, false)) {
            int page_of = 0, loaded = -1;
            for (int t = p.t0; ok && t < p.t1; ++t, ++it) {
                if (loaded < 0 || t >= loaded + per_load) {   // table entries of the next 32 boxes
                    loaded = t;
                    const int key = t * kTileKeys + lane * R;
                    page_of = key < p.seen ? __ldg(a.page_table + (long long)p.b * a.table_stride + key / a.page_size) : -1;
                }
                const int s = it & 1, key0 = t * kTileKeys;
                const unsigned use = (unsigned)it >> 1;
                const int src = min((t - loaded) * nb + lane, 31);
                const int page = __shfl_sync(0xffffffffu, page_of, src), key = key0 + lane * R;
                const bool mine = lane < nb, live = mine && key < p.seen, good = live && page >= 0 && page < a.num_pages;
                if (live && !good && a.status) atomicOr(a.status, kStatusBadPage);
                const unsigned long long bits = (good ? (R == 64 ? ~0ull : (1ull << R) - 1) << (lane * R & 63) : 0ull);
                unsigned long long m = (unsigned long long)__reduce_or_sync(0xffffffffu, (unsigned)(bits >> 32)) << 32 |
                                       __reduce_or_sync(0xffffffffu, (unsigned)bits);
                if (p.seen - key0 < 64) m &= (1ull << (p.seen - key0)) - 1;
                const int y = key % a.page_size, z = good ? page : a.num_pages;   // z = num_pages: outside, read as zeros
                const uint32_t dst = base + kKvOff + s * kTileBytes + lane * R * 128;
#pragma unroll
                for (int g = 0; g < kGroups; ++g) {
                    if (use > 0 && !bar_wait_warp(&sh.kv_empty[s][g], (use - 1) & 1)) {
                        ok = false;
                        issued = g;
                        break;
                    }
                    if (lane == 0) {
                        if (g == 0) sh.mask[s] = m;
                        bar_expect(&sh.kv_full[s][g], g < 4 ? 2 * kChunkBytes : kChunkBytes);
                    }
                    __syncwarp();
                    if (mine) {
                        tma_load_3d(dst + 2 * g * kChunkBytes, &map, 2 * g * 64, y, z, &sh.kv_full[s][g]);
                        if (g < 4) tma_load_3d(dst + (2 * g + 1) * kChunkBytes, &map, (2 * g + 1) * 64, y, z, &sh.kv_full[s][g]);
                    }
                    __syncwarp();
                }
            }
        }
        // nothing is owed to this CTA's memory when it leaves: neither the releases of the last tiles nor, after a wait that
        // ran out, copies in flight
        for (int n = max(it - 2, 0); n < it; ++n)
            for (int g = 0; g < (n == it - 1 ? issued : kGroups); ++g)
                if (!ok || !bar_wait_warp(&sh.kv_empty[n & 1][g], (n >> 1) & 1)) {
                    ok = false;
                    bar_wait_warp(&sh.kv_full[n & 1][g], (n >> 1) & 1);
                }
    } else if (warp == 1) {
        // ── MMAs ──
        int it = 0, pieces = 0;
        const uint32_t q = base + kQOff, pb = base + kPOff;
        auto scores = [&](int n, bool last) {      // S of tile n
            const int s = n & 1;
            const uint32_t c = base + kKvOff + s * kTileBytes, d = tmem + kSCol + 64 * s;
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                if (!bar_wait_warp(&sh.kv_full[s][g], (n >> 1) & 1)) return false;
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < (g < 4 ? 8 : 4); ++k) {
                        const uint32_t off = (2 * g + (k >> 2)) * kChunkBytes + (k & 3) * 32;
                        umma_ss(d, desc_k(q + off), desc_k(c + off), kIdescS<T>, (uint32_t)(g + k > 0));
                    }
                }
                __syncwarp();
            }
            if (elect_one()) {
                umma_commit(&sh.s_full[s]);
                umma_commit(&sh.kv_empty[s][4]);
                if (last) umma_commit(&sh.q_empty);
            }
            __syncwarp();
            return true;
        };
        while (ok && walk.next(p, false)) {
            const int n = p.t1 - p.t0;
            ok = bar_wait_warp(&sh.q_full, pieces & 1);
            tc_fence_after();
            ok = ok && scores(it, n == 1);
            for (int i = 0; ok && i < n; ++i, ++it) {
                if (i + 1 < n) ok = scores(it + 1, i + 2 == n);
                ok = ok && bar_wait_warp(&sh.p_full, it & 1);
                if (!ok) break;
                tc_fence_after();
                const uint32_t c = base + kKvOff + (it & 1) * kTileBytes;
                if (elect_one()) {
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            umma_ss(tmem + 64 * g, desc_mn(c + 2 * g * kChunkBytes + k * 2048), desc_k(pb + k * 32), kIdescO<T>, (uint32_t)(i + k > 0));
                        umma_commit(&sh.kv_empty[it & 1][g]);
                    }
                    umma_commit(&sh.pv_done);
                }
                __syncwarp();
            }
            ++pieces;
        }
        if (!ok) {   // the MMAs that were issued have to be through before the tensor memory is freed
            if (elect_one()) umma_commit(&sh.drain);
            __syncwarp();
            bar_wait_warp(&sh.drain, 0);
        }
    } else if (warp < 4) {
        // ── Q of a piece: 64 rows, zeros behind the last one ──
        const int ltid = tid - 64;
        int pieces = 0;
        while (ok && walk.next(p, false)) {
            if (pieces > 0) ok = bar_wait(&sh.q_empty, (pieces - 1) & 1);
            if (!ok) break;
            const T* q = (const T*)a.q + (long long)p.b * a.q_len * a.q_token;
#pragma unroll 4
            for (int i = ltid; i < kTileRows * (kLatentRow / 8); i += 64) {
                const int r = i / (kLatentRow / 8), c = i - r * (kLatentRow / 8), row = p.rb * kTileRows + r;
                const bool live = row < rows_all;
                const int j = live ? row / a.heads : 0, h = live ? row - j * a.heads : 0;
                const uint32_t dst = base + kQOff + (c >> 3) * kChunkBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(q + j * a.q_token + h * a.q_head + c * 8), "r"(live ? 16 : 0)
                             : "memory");
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            proxy_fence();
            bar_arrive(&sh.q_full);
            ++pieces;
        }
        if (ok && pieces > 0) ok = bar_wait(&sh.q_empty, (pieces - 1) & 1);
    } else {
        // ── softmax and results ──
        // (a thread whose wait ran out goes on to the next common barrier, where all of them leave together)
        const int w = warp & 3, r0 = 16 * w + (lane >> 2), r1 = r0 + 8, c0 = 2 * (lane & 3);
        const uint32_t quarter = (uint32_t)(32 * w) << 16;
        const int stid = tid - 128;
        if (stid == 0) a.owner[blockIdx.x] = make_int4(0, 0, 0, 0);
        int it = 0;
        while (ok && walk.next(p, true)) {
            const int len = max(__ldg(a.seq_lens + p.b), 0);
            const long long token0 = (long long)p.b * a.q_len;
            if (stid == 0 && len > a.max_pages * a.page_size && a.status) atomicOr(a.status, kStatusBadPage);
            if (p.tiles == 0) {      // no row of the block sees a key
                const int n = min(kTileRows, rows_all - p.rb * kTileRows);
                for (int r = w; r < n; r += 4) {
                    const int row = p.rb * kTileRows + r, j = row / a.heads, h = row - j * a.heads;
                    uint4* o = reinterpret_cast<uint4*>((T*)a.out + (token0 + j) * a.out_token + h * a.out_head);
                    o[lane] = o[lane + 32] = make_uint4(0, 0, 0, 0);
                    if (lane == 0 && a.lse) a.lse[(token0 + j) * a.heads + h] = -INFINITY;
                }
                continue;
            }
            const int j0 = (p.rb * kTileRows + r0) / a.heads, j1 = (p.rb * kTileRows + r1) / a.heads;
            const int seen0 = min(len - a.q_len + j0 + 1, p.seen), seen1 = min(len - a.q_len + j1 + 1, p.seen);
            const int seen_all = min(len - a.q_len + p.rb * kTileRows / a.heads + 1, p.seen);    // keys that every row sees
            float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
            for (int t = p.t0; t < p.t1; ++t, ++it) {
                const int s = it & 1, key0 = t * kTileKeys;
                ok = ok && bar_wait(&sh.kv_full[s][0], (it >> 1) & 1) && bar_wait(&sh.s_full[s], (it >> 1) & 1);
                __syncwarp();
                const unsigned long long mask = sh.mask[s];
                tc_fence_after();
                uint32_t raw[32];
                tmem_ld_16x64(tmem + kSCol + 64 * s + quarter, raw);
                tmem_ld_wait();
                float v[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(raw[i]) * a.scale_log2;
                if (mask != ~0ull || key0 + kTileKeys > seen_all) {
                    // (values in masked places may be anything: they are replaced, not multiplied)
                    const unsigned long long k0 = seen0 - key0 >= 64 ? mask : seen0 > key0 ? mask & ((1ull << (seen0 - key0)) - 1) : 0ull;
                    const unsigned long long k1 = seen1 - key0 >= 64 ? mask : seen1 > key0 ? mask & ((1ull << (seen1 - key0)) - 1) : 0ull;
#pragma unroll
                    for (int x = 0; x < 8; ++x)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            if (!(k0 >> (8 * x + c0 + e) & 1)) v[4 * x + e] = -INFINITY;
                            if (!(k1 >> (8 * x + c0 + e) & 1)) v[4 * x + 2 + e] = -INFINITY;
                        }
                }
                float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    x0 = fmaxf(x0, fmaxf(v[4 * x], v[4 * x + 1]));
                    x1 = fmaxf(x1, fmaxf(v[4 * x + 2], v[4 * x + 3]));
                }
#pragma unroll
                for (int x = 1; x < 4; x <<= 1) {
                    x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, x));
                    x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, x));
                }
                float f0 = 1.f, f1 = 1.f;
                if (x0 > m0 + kLazy) {
                    f0 = m0 == -INFINITY ? 1.f : ex2(m0 - x0);
                    m0 = x0;
                    l0 *= f0;
                }
                if (x1 > m1 + kLazy) {
                    f1 = m1 == -INFINITY ? 1.f : ex2(m1 - x1);
                    m1 = x1;
                    l1 *= f1;
                }
                if ((lane & 3) == 0) {
                    sh.factor[s][r0] = f0;
                    sh.factor[s][r1] = f1;
                }
                const bool rescale = softmax_any(f0 != 1.f || f1 != 1.f || !ok);
                if (rescale && softmax_any(!ok)) {
                    ok = false;
                    break;
                }
                const float n0 = m0 == -INFINITY ? 0.f : m0, n1 = m1 == -INFINITY ? 0.f : m1;
                float s0 = 0.f, s1 = 0.f;
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    v[4 * x] = ex2(v[4 * x] - n0);
                    v[4 * x + 1] = ex2(v[4 * x + 1] - n0);
                    v[4 * x + 2] = ex2(v[4 * x + 2] - n1);
                    v[4 * x + 3] = ex2(v[4 * x + 3] - n1);
                    s0 += v[4 * x] + v[4 * x + 1];
                    s1 += v[4 * x + 2] + v[4 * x + 3];
                }
                l0 += s0;
                l1 += s1;
                // P and O belong to the product of the tile before until that is through
                if (it > 0) ok = bar_wait(&sh.pv_done, (it - 1) & 1);
                __syncwarp();
                if (rescale && t > p.t0) {
                    tc_fence_after();
#pragma unroll 1
                    for (int x = 0; x < 8; ++x) {
                        uint32_t o[32];
                        tmem_ld_32x32(tmem + 32 * x + quarter, o);
                        tmem_ld_wait();
                        const float4* f = reinterpret_cast<const float4*>(&sh.factor[s][32 * (x & 1)]);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float4 y = f[i];
                            o[4 * i] = __float_as_uint(__uint_as_float(o[4 * i]) * y.x);
                            o[4 * i + 1] = __float_as_uint(__uint_as_float(o[4 * i + 1]) * y.y);
                            o[4 * i + 2] = __float_as_uint(__uint_as_float(o[4 * i + 2]) * y.z);
                            o[4 * i + 3] = __float_as_uint(__uint_as_float(o[4 * i + 3]) * y.w);
                        }
                        tmem_st_32x32(tmem + 32 * x + quarter, o);
                    }
                    tmem_st_wait();
                }
                unsigned char* pr = smem + kPOff;
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    *reinterpret_cast<uint32_t*>(pr + r0 * 128 + ((x ^ (r0 & 7)) << 4) + 2 * c0) = pack2<T>(v[4 * x], v[4 * x + 1]);
                    *reinterpret_cast<uint32_t*>(pr + r1 * 128 + ((x ^ (r1 & 7)) << 4) + 2 * c0) = pack2<T>(v[4 * x + 2], v[4 * x + 3]);
                }
                if (p.seen - key0 < kTileKeys && p.seen % a.box_rows) {
                    // rows behind the sequence came with its last box: their weights are 0, and 0 times what lies there has to be 0
                    const int first = p.seen - key0, n = (kTileKeys - first) * 8;
                    for (int c = 0; c < 8; ++c)
                        for (int i = stid; i < n; i += kSoftmaxThreads)
                            *reinterpret_cast<uint4*>(smem + kKvOff + s * kTileBytes + c * kChunkBytes + first * 128 + i * 16) = make_uint4(0, 0, 0, 0);
                }
                proxy_fence();
                tc_fence_before();
                bar_arrive(&sh.p_full);
            }
            ok = ok && bar_wait(&sh.pv_done, (it - 1) & 1);
            ok = !softmax_any(!ok);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int x = 1; x < 4; x <<= 1) {
                l0 += __shfl_xor_sync(0xffffffffu, l0, x);
                l1 += __shfl_xor_sync(0xffffffffu, l1, x);
            }
            const bool whole = p.t0 == 0 && p.t1 == p.tiles;
            const int slot = 2 * blockIdx.x + (p.t0 == 0 ? 1 : 0);
            if ((lane & 3) == 0) {
                const int row0 = p.rb * kTileRows + r0, row1 = row0 + 8;
                if (whole) {
                    sh.inv[r0] = l0 == 0.f ? 0.f : 1.f / l0;
                    sh.inv[r1] = l1 == 0.f ? 0.f : 1.f / l1;
                    if (a.lse) {
                        if (row0 < rows_all) a.lse[token0 * a.heads + row0] = l0 == 0.f ? -INFINITY : (m0 + log2f(l0)) * 0.69314718055994530942f;
                        if (row1 < rows_all) a.lse[token0 * a.heads + row1] = l1 == 0.f ? -INFINITY : (m1 + log2f(l1)) * 0.69314718055994530942f;
                    }
                } else {
                    a.part_ml[slot * kTileRows + r0] = make_float2(m0, l0);
                    a.part_ml[slot * kTileRows + r1] = make_float2(m1, l1);
                }
            }
            if (!whole && p.t0 == 0 && stid == 0) {
                // the share that holds the item's last tile: the smallest s with total (s + 1) / shares beyond it
                const long long behind = p.prefix + p.tiles;
                const int last = (int)((behind * plan.shares + plan.total - 1) / plan.total) - 1;
                a.owner[blockIdx.x] = make_int4(p.b, p.rb, last - plan.share + 1, 0);
            }
            softmax_sync();
            const int d0 = 32 * w + lane;
            if (whole) {
                const int n = min(kTileRows, rows_all - p.rb * kTileRows);
#pragma unroll 1
                for (int x = 0; x < 8; ++x) {
                    uint32_t o[32];
                    tmem_ld_32x32(tmem + 32 * x + quarter, o);
                    tmem_ld_wait();
                    const int rb = 32 * (x & 1);
                    int j = (p.rb * kTileRows + rb) / a.heads, h = p.rb * kTileRows + rb - j * a.heads;
                    T* out = (T*)a.out + 128 * (x >> 1) + d0;
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        if (rb + i < n) out[(token0 + j) * a.out_token + h * a.out_head] = from_float<T>(__uint_as_float(o[i]) * sh.inv[rb + i]);
                        if (++h == a.heads) { h = 0; ++j; }
                    }
                }
            } else {
                float* out = a.part_o + slot * kPartFloats + d0;
#pragma unroll 1
                for (int x = 0; x < 8; ++x) {
                    uint32_t o[32];
                    tmem_ld_32x32(tmem + 32 * x + quarter, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) out[(32 * (x & 1) + i) * kRank + 128 * (x >> 1)] = __uint_as_float(o[i]);
                }
            }
            tc_fence_before();
        }
    }
    if (!ok && lane == 0 && a.status) atomicOr(a.status, 4 /* VIB3_STATUS_TIMEOUT */);
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kTmemCols) : "memory");
    }
}

// Adds up the parts of the sequences that several CTAs shared.  A block takes rows (owner, row) in turn: 128 threads cover the 512
// values, four such teams take every fourth part.  Parts of an owner c lie in its second slot and in the first slots of the CTAs after it in its lane.
constexpr int kCombineTeams = 4;

template <typename T>
__global__ void __launch_bounds__(kCombineTeams * 128) latent_combine_kernel(const AttentionArgs a, int grid) {
    __shared__ float weight[kMaxGrid];
    __shared__ float4 sums[kCombineTeams - 1][128];
    pdl_enter();
    const int tid = threadIdx.x, team = tid >> 7, x = tid & 127;
    for (int i = blockIdx.x; i < grid * kTileRows; i += gridDim.x) {
        const int c = i / kTileRows, r = i % kTileRows;
        const int4 own = a.owner[c];
        const int row = own.y * kTileRows + r;
        if (own.z == 0 || row >= a.q_len * a.heads) continue;
        const int parts = own.z;
        const long long token = (long long)own.x * a.q_len + row / a.heads;
        const int h = row % a.heads;
        if (tid < 32) {
            float m = -INFINITY, l = 0.f;
            for (int k = tid; k < parts; k += 32) m = fmaxf(m, a.part_ml[(2 * (c + k * a.lanes) + (k == 0)) * kTileRows + r].x);
#pragma unroll
            for (int y = 16; y; y >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, y));
            for (int k = tid; k < parts; k += 32) {
                const float2 ml = a.part_ml[(2 * (c + k * a.lanes) + (k == 0)) * kTileRows + r];
                const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - m);
                weight[k] = f;
                l = fmaf(f, ml.y, l);
            }
#pragma unroll
            for (int y = 16; y; y >>= 1) l += __shfl_xor_sync(0xffffffffu, l, y);
            const float inv = l == 0.f ? 0.f : 1.f / l;
            __syncwarp();
            for (int k = tid; k < parts; k += 32) weight[k] *= inv;
            if (tid == 0 && a.lse) a.lse[token * a.heads + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994530942f;
        }
        __syncthreads();
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int k = team; k < parts; k += kCombineTeams) {
            const float f = weight[k];
            const float4 v = *reinterpret_cast<const float4*>(a.part_o + (2 * (c + k * a.lanes) + (k == 0)) * kPartFloats + r * kRank + 4 * x);
            o.x = fmaf(f, v.x, o.x); o.y = fmaf(f, v.y, o.y); o.z = fmaf(f, v.z, o.z); o.w = fmaf(f, v.w, o.w);
        }
        if (team) sums[team - 1][x] = o;
        __syncthreads();
        if (team == 0) {
#pragma unroll
            for (int t = 0; t < kCombineTeams - 1; ++t) {
                const float4 v = sums[t][x];
                o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
            }
            uint2 b;
            b.x = pack2<T>(o.x, o.y);
            b.y = pack2<T>(o.z, o.w);
            *reinterpret_cast<uint2*>((T*)a.out + token * a.out_token + h * a.out_head + 4 * x) = b;
        }
    }
}

namespace {

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                             const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn tensor_map_encoder() {
    static EncodeFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess) {
            p = nullptr;
            (void)cudaGetLastError();
        }
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}

constexpr size_t kOwnerBytes = kMaxGrid * sizeof(int4), kMlBytes = 2 * (size_t)kMaxGrid * kTileRows * sizeof(float2);
constexpr size_t kAttWorkspace = kOwnerBytes + kMlBytes + 2 * (size_t)kMaxGrid * kPartFloats * sizeof(float);

template <typename T>
int launch_attention(const CUtensorMap& map, const AttentionArgs& a, int grid, cudaStream_t st) {
    cudaError_t e = cudaFuncSetAttribute(latent_attention_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kAttSmem);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return (int)e;
    }
    const int r = launch_latent(latent_attention_kernel<T>, dim3((unsigned)grid), kAttThreads, kAttSmem, st, map, a);
    if (r) return r;
    return launch_latent(latent_combine_kernel<T>, dim3((unsigned)(4 * grid)), kCombineTeams * 128, 0, st, a, grid);
}

}  // namespace

}  // namespace vib3

using namespace vib3;

extern "C" size_t vib3_latent_attention_workspace_bytes(void) { return kAttWorkspace; }

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
        page_size > (1 << 20) || max_pages_per_seq <= 0 || (long long)max_pages_per_seq * page_size > 0x7fffff00 ||
        (long long)batch * q_len > (1 << 20))
        return VIB3_ERR_COUNT;
    // (a tensor map's strides are below 2^40 bytes)
    if (row_stride < kLatentRow || page_stride < row_stride * (page_size - 1) + kLatentRow || page_stride >= (1ll << 38) || q_token_stride < 0 ||
        q_head_stride < 0 || (batch > 1 && table_stride < max_pages_per_seq) || (heads > 1 && out_head_stride < kRank) ||
        ((long long)batch * q_len > 1 && out_token_stride < kRank))
        return VIB3_ERR_SHAPE;
    if (((uintptr_t)q & 15) || ((uintptr_t)cache & 15) || ((uintptr_t)out & 15) || ((uintptr_t)workspace & 15) || q_token_stride % 8 ||
        q_head_stride % 8 || page_stride % 8 || row_stride % 8 || out_token_stride % 8 || out_head_stride % 8)
        return VIB3_ERR_ALIGN;
    if (workspace_bytes < kAttWorkspace) return VIB3_ERR_CAPACITY;
    if (batch == 0 || q_len == 0) return VIB3_OK;
    const EncodeFn encode = tensor_map_encoder();
    if (!encode) return VIB3_ERR_UNSUPPORTED;

    AttentionArgs a;
    a.q = q; a.q_token = q_token_stride; a.q_head = q_head_stride;
    a.page_size = page_size; a.num_pages = (int)num_pages;
    a.box_rows = page_size % 64 == 0 ? 64 : page_size % 32 == 0 ? 32 : page_size % 16 == 0 ? 16 : 8;
    a.page_table = page_table; a.table_stride = table_stride; a.max_pages = max_pages_per_seq;
    a.seq_lens = seq_lens; a.batch = batch; a.q_len = q_len; a.heads = heads;
    a.scale_log2 = scale * 1.4426950408889634074f;
    a.out = out; a.out_token = out_token_stride; a.out_head = out_head_stride;
    a.lse = lse_or_null; a.status = status;
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    a.owner = reinterpret_cast<int4*>(ws);
    a.part_ml = reinterpret_cast<float2*>(ws + kOwnerBytes);
    a.part_o = reinterpret_cast<float*>(ws + kOwnerBytes + kMlBytes);
    const int blocks = (int)(((long long)q_len * heads + kTileRows - 1) / kTileRows);
    const int sms = sm_count() < kMaxGrid ? sm_count() : kMaxGrid;
    a.lanes = blocks <= 8 ? blocks : 1;
    a.blocks_per_lane = blocks / a.lanes;
    if ((long long)batch * a.blocks_per_lane > 0x7fffffff) return VIB3_ERR_COUNT;
    a.min_tiles = 2;
    const int grid = sms / a.lanes * a.lanes;

    CUtensorMap map;
    const cuuint64_t dims[3] = {(cuuint64_t)kLatentRow, (cuuint64_t)page_size, (cuuint64_t)num_pages};
    const cuuint64_t strides[2] = {(cuuint64_t)row_stride * 2, (cuuint64_t)page_stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)a.box_rows, 1}, one[3] = {1, 1, 1};
    if (encode(&map, dtype == L_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(cache), dims, strides,
               box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return VIB3_ERR_SHAPE;
    return dtype == L_F16 ? launch_attention<__half>(map, a, grid, (cudaStream_t)stream)
                          : launch_attention<__nv_bfloat16>(map, a, grid, (cudaStream_t)stream);
}
