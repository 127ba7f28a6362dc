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
constexpr int kQOff = 0, kKvOff = kTileBytes, kPOff = 8 * kChunkBytes /* in a tile */, kMiscOff = 3 * kTileBytes;
constexpr int kAttThreads = 384;                          // copies, MMAs, two warps for Q, eight for the softmax and the results
constexpr int kSoftmaxThreads = 256;
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
    uint64_t kv_full[2], kv_empty[2][kGroups];
    uint64_t s_full[2], p_full[2], pv_done[2], q_full, q_empty, drain;
    unsigned long long mask[2];            // keys of the tile that count
    alignas(16) float factor[kTileRows];
    float team[2][kTileRows];              // what the two softmax teams have of a row: maximum, sum
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
// One look, without waiting; the warp's lanes agree.
__device__ __forceinline__ bool bar_test(uint64_t* bar, unsigned parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return __all_sync(0xffffffffu, ok != 0);
}
constexpr unsigned kIdleLimit = 1u << 26;   // looks without progress (each some 50 cycles: about two seconds)
// The same for a whole warp, whose lanes have to agree (they meet again in warp-wide instructions).
__device__ __forceinline__ bool bar_wait_warp(uint64_t* bar, unsigned parity) { return __all_sync(0xffffffffu, bar_wait(bar, parity)); }
// 16 bytes global -> shared, zeros where !live
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
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
// Shared-memory operands with 128-byte swizzle.  K-major: rows of 128 bytes, eight of them 1024 bytes.  MN-major: 64 values
// contiguous per key, eight keys 1024 bytes, the next 64 values a chunk further.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k(uint32_t addr) { return ((addr & 0x3FFFF) >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn(uint32_t addr) { return ((addr & 0x3FFFF) >> 4) | ((uint32_t)(kChunkBytes >> 4) << 16); }
// A value that is the same in all lanes, told to the compiler: an MMA takes its operands from uniform registers, and with
// operands that it had to move there one by one an MMA of this kernel cost 85 cycles instead of the pipe's 32 or 48.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }
// Operands by the low words of their descriptors (the address); the high words are constants.
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}"
                 ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(kDescHigh) : "memory");
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

template <typename T> constexpr uint32_t kFormat = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
template <typename T> constexpr uint32_t kIdescS = (1u << 4) | (kFormat<T> << 7) | (kFormat<T> << 10) | (64u / 8 << 17) | (64u / 16 << 24);
template <typename T> constexpr uint32_t kIdescO = (1u << 4) | (kFormat<T> << 7) | (kFormat<T> << 10) | (1u << 15) | (64u / 8 << 17) | (128u / 16 << 24);

// 16 lanes x 32 columns: thread t has columns 8 x + 2 (t & 3) + {0, 1} of lane t / 4 (registers 4 x, 4 x + 1) and of lane t / 4 + 8.
__device__ __forceinline__ void tmem_ld_16x32(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr) : "memory");
}
// 32 lanes x 32 columns, a lane per thread.
__device__ __forceinline__ void tmem_ld_32x32(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr) : "memory");
}

__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}

// This CTA's place on its lane's line of tiles.  All threads.  Up to kAttThreads items are read once and stay in registers.
__device__ __forceinline__ void make_plan(const AttentionArgs& a, AttShared& sh) {
    constexpr int kWarps = kAttThreads / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row_lane = a.lanes == 1 ? 0 : blockIdx.x % a.lanes, share = a.lanes == 1 ? blockIdx.x : blockIdx.x / a.lanes, items = item_count(a);
    const int most = a.lanes == 1 ? gridDim.x : gridDim.x / a.lanes;
    Piece p;
    auto tiles_of = [&](int i) {
        if (i >= items) return 0;
        item_of(a, row_lane, i, p);
        return p.tiles;
    };
    // inclusive sum over the block's threads; `sum` receives the total
    auto block_scan = [&](long long v, long long& sum) {
#pragma unroll
        for (int m = 1; m < 32; m <<= 1) {
            const long long o = __shfl_up_sync(0xffffffffu, v, m);
            if (lane >= m) v += o;
        }
        __syncthreads();
        if (lane == 31) sh.warp_sum[warp] = v;
        __syncthreads();
        sum = 0;
        long long before = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w == warp) before = sum;
            sum += sh.warp_sum[w];
        }
        return before + v;
    };
    const int first_tiles = tiles_of(tid);
    long long mine = first_tiles, chunk, total;
    for (int i = tid + kAttThreads; i < items; i += kAttThreads) mine += tiles_of(i);
    long long incl = block_scan(mine, total);
    const int shares = (int)max(1ll, min((long long)most, (total + a.min_tiles - 1) / a.min_tiles));
    const bool idle = share >= shares;
    // (a 64-bit division is a subroutine of some hundred instructions)
    auto cut = [&](int k) {
        return total <= 0x7fffffff / kMaxGrid ? (long long)((unsigned)total * (unsigned)k / (unsigned)shares) : total * k / shares;
    };
    const long long begin = idle ? total : cut(share), end = idle ? total : cut(share + 1);
    if (tid == 0) {
        sh.plan.begin = begin; sh.plan.end = end; sh.plan.total = total;
        sh.plan.lane = row_lane; sh.plan.share = share; sh.plan.shares = shares;
        if (idle) {
            sh.plan.item = items;
            sh.plan.prefix = total;
        }
    }
    if (idle) return;
    // the first item that begins at `begin` or reaches beyond it
    long long base = 0;
    for (int i0 = 0; i0 < items; i0 += kAttThreads) {
        const int i = i0 + tid, tiles = i0 == 0 ? first_tiles : tiles_of(i);
        if (items > kAttThreads) incl = block_scan(tiles, chunk);
        else chunk = total;
        const long long pre = base + incl - tiles;
        // of those that qualify the first one: nothing before it begins at `begin`, and what comes before does not reach beyond
        if (i < items && pre <= begin && (pre == begin || pre + tiles > begin)) {
            bool first = true;
            if (pre == begin && i > 0) {   // an item before this one with the same beginning (no tiles) comes first
                item_of(a, row_lane, i - 1, p);
                first = p.tiles > 0;
            }
            if (first) {
                sh.plan.item = i;
                sh.plan.prefix = pre;
            }
        }
        base += chunk;
        if (base > begin) break;
    }
}

template <typename T>
__global__ void __launch_bounds__(kAttThreads, 1) latent_attention_kernel(const __grid_constant__ CUtensorMap map, const AttentionArgs a) {
    extern __shared__ __align__(1024) unsigned char smem[];
    AttShared& sh = *reinterpret_cast<AttShared*>(smem + kMiscOff);
    const uint32_t base = smem_u32(smem);
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    if (tid == 0) {
        for (int s = 0; s < 2; ++s) {
            bar_init(&sh.kv_full[s], 1);
            for (int g = 0; g < kGroups; ++g) bar_init(&sh.kv_empty[s][g], 1);
            bar_init(&sh.s_full[s], 1);
            bar_init(&sh.p_full[s], kSoftmaxThreads);
            bar_init(&sh.pv_done[s], 1);
        }
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
    const uint32_t tmem = uniform(sh.tmem);
    const Plan& plan = sh.plan;
    const int rows_all = a.q_len * a.heads;
    Walk walk(a, plan);
    Piece p;
    bool ok = (base & 1023) == 0;   // the swizzle is a function of the address

    if (warp == 0) {
        // ── copies: the tiles of C, in boxes of box_rows rows that lie in one page ──
        const int R = a.box_rows, nb = kTileKeys / R, per_load = 32 / nb;
        int it = 0;
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
                        // the tile's remaining bytes will not come: what was requested is waited for below, this tile cannot be
                        ok = false;
                        break;
                    }
                    if (g == 0) {
                        if (lane == 0) {
                            sh.mask[s] = m;
                            bar_expect(&sh.kv_full[s], kTileBytes);
                        }
                        __syncwarp();
                    }
                    if (mine) {
                        tma_load_3d(dst + 2 * g * kChunkBytes, &map, 2 * g * 64, y, z, &sh.kv_full[s]);
                        if (g < 4) tma_load_3d(dst + (2 * g + 1) * kChunkBytes, &map, (2 * g + 1) * 64, y, z, &sh.kv_full[s]);
                    }
                    __syncwarp();
                }
            }
        }
        // Nothing is owed to this CTA's memory when it leaves: the releases of the last tiles arrive, or, after a wait that ran out,
        // the copies in flight do (the newest tile's barrier may lack bytes that were never requested: that wait gives up).
        for (int n = max(it - 2, 0); n < it; ++n)
            for (int g = 0; g < kGroups; ++g)
                if (!ok || !bar_wait_warp(&sh.kv_empty[n & 1][g], (n >> 1) & 1)) {
                    ok = false;
                    bar_wait_warp(&sh.kv_full[n & 1], (n >> 1) & 1);
                    break;
                }
    } else if (warp == 1) {
        // ── MMAs ──
        // Two walks over the same tiles, S at most two tiles ahead of O (its two buffers).  Whatever has its operands goes next, O
        // first, since only O gives shared memory back: with S(i + 1) always before O(i), O waited for the load of tile i + 1,
        // which waits for the room of tile i - 1, and a tile took 4100 cycles.
        Walk walk_o(a, plan);
        Piece po;
        bool more_s = ok && walk.next(p, false), more_o = ok && walk_o.next(po, false);
        int ns = 0, ts = p.t0, q_pieces = 0;              // next S: tile count, tile of the item, pieces whose Q was read
        int no = 0, to = po.t0;                           // next O
        bool q_ready = false;
        unsigned idle = 0;
        while (more_o) {
            if (no < ns && bar_test(&sh.p_full[no & 1], (no >> 1) & 1)) {
                tc_fence_after();
                const int st = (int)uniform((uint32_t)no & 1);
                const uint32_t c = uniform(base + kKvOff + st * kTileBytes), v = desc_mn(c), pk = desc_k(c + kPOff), acc = uniform(to > po.t0);
                if (elect_one()) {
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            umma_ss(tmem + 64 * g, v + (2 * g * kChunkBytes + k * 2048) / 16, pk + k * 2, kIdescO<T>, k > 0 ? 1u : acc);
                        umma_commit(&sh.kv_empty[st][g]);
                    }
                    umma_commit(&sh.kv_empty[st][kGroups - 1]);
                    umma_commit(&sh.pv_done[st]);
                }
                __syncwarp();
                ++no;
                if (++to == po.t1) {
                    more_o = walk_o.next(po, false);
                    to = po.t0;
                }
                idle = 0;
                continue;
            }
            if (more_s && ns < no + 2) {
                if (!q_ready && bar_test(&sh.q_full, q_pieces & 1)) q_ready = true;
                if (q_ready && bar_test(&sh.kv_full[ns & 1], (ns >> 1) & 1)) {
                    tc_fence_after();
                    const bool piece_end = ts + 1 == p.t1;
                    const int st = (int)uniform((uint32_t)ns & 1);
                    const uint32_t d = uniform(tmem + kSCol + 64 * st), qd = uniform(desc_k(base + kQOff)), cd = uniform(desc_k(base + kKvOff + st * kTileBytes));
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < 4 * kChunks; ++k)
                            umma_ss(d, qd + (k >> 2) * kChunkBytes / 16 + (k & 3) * 2, cd + (k >> 2) * kChunkBytes / 16 + (k & 3) * 2, kIdescS<T>, k > 0);
                        umma_commit(&sh.s_full[st]);
                        if (piece_end) umma_commit(&sh.q_empty);
                    }
                    __syncwarp();
                    ++ns;
                    ++ts;
                    if (piece_end) {
                        q_ready = false;
                        ++q_pieces;
                        more_s = walk.next(p, false);
                        ts = p.t0;
                    }
                    idle = 0;
                    continue;
                }
            }
            if (++idle > kIdleLimit) {
                ok = false;
                break;
            }
        }
        if (!ok) {   // the MMAs that were issued have to be through before the tensor memory is freed
            if (elect_one()) umma_commit(&sh.drain);
            __syncwarp();
            bar_wait_warp(&sh.drain, 0);
        }
    } else if (warp < 4) {
        // ── Q of a piece: 64 rows, zeros behind the last one ──
        int pieces = 0;
        while (ok && walk.next(p, false)) {
            if (pieces > 0) ok = bar_wait_warp(&sh.q_empty, (pieces - 1) & 1);
            if (!ok) break;
            const long long token0 = (long long)p.b * a.q_len;
            // A warp takes every second row; lane i works out the address of its i-th (a division per 16 bytes: 8 us per piece).
            const int row = p.rb * kTileRows + 2 * lane + (warp & 1), j = row / a.heads, h = row - j * a.heads;
            const long long at = row < rows_all ? (token0 + j) * a.q_token + h * a.q_head : -1;
            const uint32_t piece = (uint32_t)(lane & 7), chunk = base + kQOff + (lane >> 3) * kChunkBytes;
#pragma unroll 8
            for (int i = 0; i < kTileRows / 2; ++i) {
                const long long off = __shfl_sync(0xffffffffu, at, i);
                const bool live = off >= 0;
                const T* src = (const T*)a.q + (live ? off : 0) + lane * 8;
                const int r = 2 * i + (warp & 1);
                const uint32_t dst = chunk + r * 128 + ((piece ^ (r & 7)) << 4);
                cp_async16(dst, src, live);
                cp_async16(dst + 4 * kChunkBytes, src + 256, live);
                if (lane < 8) cp_async16(dst + 8 * kChunkBytes, src + 512, live);
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            proxy_fence();
            bar_arrive(&sh.q_full);
            ++pieces;
        }
        if (ok && pieces > 0) ok = bar_wait(&sh.q_empty, (pieces - 1) & 1);
    } else {
        // ── softmax and results ──
        // Two teams of four warps, 32 keys each; warp w of a team has rows 16 w .. (their lanes in tensor memory), a thread two rows
        // and eight keys of each.  (A thread whose wait ran out goes on to the next common barrier, where all of them leave.)
        const int team = (warp - 4) >> 2, w = warp & 3, r0 = 16 * w + (lane >> 2), r1 = r0 + 8, c0 = 32 * team + 2 * (lane & 3);
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
                for (int r = warp - 4; r < n; r += 8) {
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
                const unsigned parity = (unsigned)(it >> 1) & 1;
                // (the tile two before is through when this one's scores are; seen here, its phase cannot be taken for another)
                ok = ok && (it < 2 || bar_wait(&sh.pv_done[s], parity ^ 1)) && bar_wait(&sh.kv_full[s], parity) && bar_wait(&sh.s_full[s], parity);
                __syncwarp();
                const unsigned long long mask = sh.mask[s];
                tc_fence_after();
                uint32_t raw[16];
                tmem_ld_16x32(tmem + kSCol + 64 * s + 32 * team + quarter, raw);
                tmem_ld_wait();
                float v[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(raw[i]) * a.scale_log2;
                if (mask != ~0ull || key0 + kTileKeys > seen_all) {
                    // (values in masked places may be anything: they are replaced, not multiplied)
                    const unsigned long long k0 = seen0 - key0 >= 64 ? mask : seen0 > key0 ? mask & ((1ull << (seen0 - key0)) - 1) : 0ull;
                    const unsigned long long k1 = seen1 - key0 >= 64 ? mask : seen1 > key0 ? mask & ((1ull << (seen1 - key0)) - 1) : 0ull;
#pragma unroll
                    for (int x = 0; x < 4; ++x)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            if (!(k0 >> (8 * x + c0 + e) & 1)) v[4 * x + e] = -INFINITY;
                            if (!(k1 >> (8 * x + c0 + e) & 1)) v[4 * x + 2 + e] = -INFINITY;
                        }
                }
                float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    x0 = fmaxf(x0, fmaxf(v[4 * x], v[4 * x + 1]));
                    x1 = fmaxf(x1, fmaxf(v[4 * x + 2], v[4 * x + 3]));
                }
                if (softmax_any(x0 > m0 + kLazy || x1 > m1 + kLazy || !ok)) {
                    // a reference moves: the rows' maxima over both teams, then O's rows times exp2(old - new)
                    ok = !softmax_any(!ok);
                    if (!ok) break;
#pragma unroll
                    for (int x = 1; x < 4; x <<= 1) {
                        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, x));
                        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, x));
                    }
                    if ((lane & 3) == 0) {
                        sh.team[team][r0] = x0;
                        sh.team[team][r1] = x1;
                    }
                    softmax_sync();
                    x0 = fmaxf(x0, sh.team[team ^ 1][r0]);
                    x1 = fmaxf(x1, sh.team[team ^ 1][r1]);
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
                    if (team == 0 && (lane & 3) == 0) {
                        sh.factor[r0] = f0;
                        sh.factor[r1] = f1;
                    }
                    softmax_sync();
                    if (t > p.t0) {
                        ok = bar_wait(&sh.pv_done[s ^ 1], (unsigned)((it - 1) >> 1) & 1);
                        __syncwarp();
                        tc_fence_after();
#pragma unroll 1
                        for (int x = 4 * team; x < 4 * team + 4; ++x) {
                            uint32_t o[32];
                            tmem_ld_32x32(tmem + 32 * x + quarter, o);
                            tmem_ld_wait();
                            const float4* f = reinterpret_cast<const float4*>(&sh.factor[32 * (x & 1)]);
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
                }
                const float n0 = m0 == -INFINITY ? 0.f : m0, n1 = m1 == -INFINITY ? 0.f : m1;
                // P takes the place of the tile's position values, which no product reads again
                unsigned char* pr = smem + kKvOff + s * kTileBytes + kPOff + 4 * (lane & 3);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const float e0 = ex2(v[4 * x] - n0), e1 = ex2(v[4 * x + 1] - n0), e2 = ex2(v[4 * x + 2] - n1), e3 = ex2(v[4 * x + 3] - n1);
                    *reinterpret_cast<uint32_t*>(pr + r0 * 128 + (((4 * team + x) ^ (r0 & 7)) << 4)) = pack2<T>(e0, e1);
                    *reinterpret_cast<uint32_t*>(pr + r1 * 128 + (((4 * team + x) ^ (r1 & 7)) << 4)) = pack2<T>(e2, e3);
                    l0 += e0 + e1;
                    l1 += e2 + e3;
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
                bar_arrive(&sh.p_full[s]);
            }
            ok = ok && bar_wait(&sh.pv_done[(it - 1) & 1], (unsigned)((it - 1) >> 1) & 1);
            ok = !softmax_any(!ok);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int x = 1; x < 4; x <<= 1) {
                l0 += __shfl_xor_sync(0xffffffffu, l0, x);
                l1 += __shfl_xor_sync(0xffffffffu, l1, x);
            }
            if (team == 1 && (lane & 3) == 0) {
                sh.team[1][r0] = l0;
                sh.team[1][r1] = l1;
            }
            softmax_sync();
            const bool whole = p.t0 == 0 && p.t1 == p.tiles;
            const int slot = 2 * blockIdx.x + (p.t0 == 0 ? 1 : 0);
            if (team == 0 && (lane & 3) == 0) {
                const int row0 = p.rb * kTileRows + r0, row1 = row0 + 8;
                l0 += sh.team[1][r0];
                l1 += sh.team[1][r1];
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
            const int d0 = 32 * w + lane;
            if (whole) {
                softmax_sync();
                const int n = min(kTileRows, rows_all - p.rb * kTileRows);
#pragma unroll 1
                for (int x = 4 * team; x < 4 * team + 4; ++x) {
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
                for (int x = 4 * team; x < 4 * team + 4; ++x) {
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
