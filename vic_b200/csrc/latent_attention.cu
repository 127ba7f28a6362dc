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
//   S [64 rows x 64 keys]  = Q . C^T      tcgen05, M = 64, K = 576; Q stays in the SM for the whole sequence
//   P = exp(S - m)                        eight warps, from tensor memory to shared memory as 16-bit values
//   O^T [512 x 64 rows]   += C^T . P^T    tcgen05, four products with M = 128 values and N = 64 rows
// The tile of C that TMA brought once is operand of both products: K-major (its 576 values contiguous) in the first, and in the
// second, through another descriptor of the same bytes, MN-major.  With the accumulator transposed its 256 columns fill all 128
// lanes of tensor memory, so it stays there for the whole sequence, and the number of rows is the N of the MMA.
// Per tile the pipe is busy 36 x 32 + 16 x 48 = 1920 cycles, HBM's share of an SM 3270 at 1.965 GHz.  What decides is how long a tile stays in
// shared memory: load 2800 to 3500, S 1150, softmax 700, O 900 cycles.  With all of Q in shared memory there is room for two tiles
// and a tile took 3500 cycles; with six of its nine chunks in tensor memory for two and three quarters, and it takes 3200, HBM's rate.
// Measured, 64 heads, bf16, with the adding launch: 128 sequences of 4100 tokens 125 us (5.0 TB/s; 144 us when the card
// is held at its power limit), one of 131071 43 us, 32 of 1 to 16384 39 us, one of 4001 12.9 us.
#include "latent_tc.cuh"

namespace vib3 {

constexpr int kTileKeys = 64, kTileRows = 64;
constexpr int kChunks = kLatentRow / 64;                  // 9: eight of the latent, one of position values
constexpr int kTileBytes = kChunks * kChunkBytes;
// Shared memory: the part of Q that tensor memory has no room for, a ring of latent chunk pairs, places for position values (then P).
constexpr int kQTmemChunks = 6, kSlots = 11, kTiles = 3, kSlotBytes = 2 * kChunkBytes;
constexpr int kQOff = 0, kRingOff = (kChunks - kQTmemChunks) * kChunkBytes, kRopeOff = kRingOff + kSlots * kSlotBytes;
constexpr int kMiscOff = kRopeOff + kTiles * kChunkBytes;
constexpr int kAttThreads = 384;                          // copies, S, O, (none: a warp reads its quarter of tensor memory), eight warps for Q, the softmax and the results
constexpr int kSoftmaxThreads = 256;
constexpr int kTmemCols = 512, kSCol = 256, kQCol = 320;  // O^T: 4 x 64 columns, S: 64, Q: 6 x 32
static_assert(kQCol + 32 * kQTmemChunks <= kTmemCols, "tensor memory");
// The reference m of a row follows its maximum only when that has grown by more than 2^8, so that the accumulator is rescaled a few times per
// sequence instead of per tile.  The weights exp(s - m) are rounded to the operands' 16-bit type, since an MMA takes one type for both; their
// sum l has them unrounded.  A bf16 weight is off by 2^-8 of itself however small it is.  fp16 is subnormal below 2^-14 and has nothing below
// 2^-25, so there m stays 2^7 below the maximum and the row's largest weight lies between 2^7 and 2^15 (of 65504): a weight is off by 2^-11 of
// itself or 2^-32 of the largest, and tens of thousands of keys beside a dominating one keep their share.
constexpr float kLazy = 8.0f;
template <typename T> constexpr float kLead = std::is_same<T, __half>::value ? 7.0f : 0.0f;
constexpr int kMaxGrid = 160;                             // CTAs that the workspace has room for
constexpr size_t kPartFloats = (size_t)kTileRows * kRank;

// Exact n / d for 0 <= n < 2^bits (bits <= 31) by one wide multiplication: mul = ceil(2^shift / d) with shift = bits + ceil(log2 d)
// is off by less than d / 2^shift of a unit, so n * (the error) stays below 2^-s.  (A division instruction sequence is some twenty instructions,
// and this kernel's code is fetched cold at every launch.)
struct FastDiv {
    unsigned mul, shift;
    __device__ __forceinline__ int operator()(int n) const { return (int)((unsigned long long)(unsigned)n * mul >> shift); }
};

struct AttentionArgs {
    const void* q;
    long long q_token, q_head;             // strides in elements
    int page_size, box_rows;
    int num_pages;
    const int* page_table;
    int table_stride, max_pages;
    const int* seq_lens;
    int batch, q_len, heads;
    FastDiv by_heads, by_page;             // of rows (< 2^27), of keys (< 2^31)
    float scale_log2;                      // scale * log2(e)
    void* out;
    long long out_token, out_head;
    float* lse;
    int* status;
    int block_rows;                        // rows of a row block: kTileRows, or half of them
    int lanes, blocks_per_lane;            // see Plan
    int min_cost;                          // of a share
    // workspace: what a sequence's row block is made of, and two places per CTA for parts
    int4* made_of;                         // [items or grid] sequence, row block, parts (fewer than 2: nothing to add up), first CTA
    int by_item;                           // whether made_of goes by item or by the CTA that begins it
    float2* part_ml;                       // [2 grid][64] reference (log2) and sum
    float4* part_o;                        // [2 grid][4][8][8][32] x 4 rows: 64 x 512 values, not yet divided by the sum
};

// The split.  A sequence has row blocks of 64 rows, a row block as many tiles as its last row sees.  Few row blocks (lanes =
// their number): CTA = share * lanes + row block, so that the CTAs of a share read the same tiles at the same time and the cache
// comes from HBM once.  Many: one lane, and a sequence's row blocks follow one another.  Within a lane the tiles of all sequences form one line that
// is cut into equal shares whatever the lengths are; a sequence that a cut divides leaves parts that a second launch adds up.
struct Plan {
    int begin, end;                        // this CTA's tiles on the line
    int prefix, b, rb, len, seen, tiles;   // the first item: where it begins, and what item_of says of it
    int share, shares, per, rem;           // share s begins at s * per + min(s, rem)
};

struct Piece {
    int b, rb, len, seen, tiles;           // item: sequence, row block, keys of the sequence and of the block's last row, tiles
    int t0, t1;                            // this CTA's tiles of it
    int prefix;
};

// A row block costs what its tiles do and kPieceCost more (Q, the results, filling the pipe: 8000 to 10000 cycles), so on the line it begins
// with a stretch without tiles.  (Without it a CTA with the ends of several short sequences took twice the average.)
constexpr int kPieceCost = 4, kMinCost = 2;
__device__ __forceinline__ int cost_of(const Piece& p) { return p.tiles ? p.tiles + kPieceCost : 0; }

__device__ __forceinline__ int first_tile(const Plan& p, int share) { return share * p.per + min(share, p.rem); }

__device__ __forceinline__ void item_of(const AttentionArgs& a, int b, int rb, Piece& p) {
    p.b = b;
    p.rb = rb;
    const int last_row = min(a.q_len * a.heads, (rb + 1) * a.block_rows) - 1;
    p.len = max(__ldg(a.seq_lens + b), 0);
    p.seen = min(max(p.len - a.q_len + a.by_heads(last_row) + 1, 0), a.max_pages * a.page_size);
    p.tiles = (p.seen + kTileKeys - 1) / kTileKeys;
}

// The pieces of this CTA in order.  Items without tiles belong to the CTA whose share they stand in (t0 == t1).
struct Walk {
    const AttentionArgs& a;
    int b, rb, rb0, prefix, begin, end;
    bool last, known;
    const Plan& plan;
    __device__ __forceinline__ Walk(const AttentionArgs& a_, const Plan& p, int rb_first)
        : a(a_), b(p.b), rb(p.rb), rb0(rb_first), prefix(p.prefix), begin(p.begin), end(p.end), last(p.share == p.shares - 1), known(true), plan(p) {}
    __device__ __forceinline__ bool next(Piece& p, bool empty) {
#pragma unroll 1
        while (b < a.batch && (prefix < end || last)) {
            if (known) {
                p.b = b; p.rb = rb; p.len = plan.len; p.seen = plan.seen; p.tiles = plan.tiles;
                known = false;
            } else {
                item_of(a, b, rb, p);
            }
            if (++rb == rb0 + a.blocks_per_lane) {
                rb = rb0;
                ++b;
            }
            p.prefix = prefix;
            prefix += cost_of(p);
            p.t0 = max(begin - p.prefix - kPieceCost, 0);
            p.t1 = min(end - p.prefix - kPieceCost, p.tiles);
            if (p.tiles == 0 ? empty : !empty && p.t1 > p.t0) return true;
        }
        return false;
    }
};

template <typename T> constexpr uint32_t kIdescS = idesc<T>(64, 64, false, false);
template <typename T> constexpr uint32_t kIdescO = idesc<T>(128, 64, true, false);

struct AttShared {
    uint64_t kv_full[kTiles], slot_empty[kSlots], rope_empty[kTiles];
    uint64_t s_full, s_free, p_full[2], pv_done[2], q_full, drain[2];
    unsigned long long mask[kTiles];       // keys of the tile that count
    alignas(16) float factor[kTileRows];
    float team[2][kTileRows];              // what the two softmax teams have of a row: maximum, sum
    alignas(16) float inv[kTileRows];
    uint32_t tmem;
};
static_assert(kMiscOff + sizeof(AttShared) <= 227 * 1024, "shared memory of a CTA");
constexpr int kAttSmem = kMiscOff + (int)sizeof(AttShared);

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// A row's log of its sum, from the reference (log2) and the sum relative to it; a part's weight relative to the largest reference.
__device__ __forceinline__ float lse_of(float m, float l) { return l == 0.f ? -INFINITY : (m + __log2f(l)) * 0.69314718055994530942f; }
__device__ __forceinline__ float weight_of(float part, float m) { return part == -INFINITY ? 0.f : ex2(part - m); }
// 32 registers of a lane as eight groups of four: afterwards lane 4 q + s has of every group i the values that the lanes 4 q .. 4 q + 3
// had in its register s.
__device__ __forceinline__ void transpose4(uint32_t* o, int sub) {
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
#pragma unroll
        for (int e = 0; e < 4; e += 2) {      // lanes that differ in bit 0 exchange the off-diagonal registers of (e, e + 1)
            const uint32_t give = sub & 1 ? o[i + e] : o[i + e + 1], got = __shfl_xor_sync(0xffffffffu, give, 1);
            if (sub & 1) o[i + e] = got;
            else o[i + e + 1] = got;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {         // bit 1: registers (e, e + 2)
            const uint32_t give = sub & 2 ? o[i + e] : o[i + e + 2], got = __shfl_xor_sync(0xffffffffu, give, 2);
            if (sub & 2) o[i + e] = got;
            else o[i + e + 2] = got;
        }
    }
}
// Named barrier of the softmax warps; the second form tells whether any of them says so.
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kSoftmaxThreads) : "memory"); }
__device__ __forceinline__ bool softmax_any(bool v) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"((uint32_t)v), "n"(kSoftmaxThreads) : "memory");
    return r != 0;
}


// 16 lanes x 32 columns: thread t has columns 8 x + 2 (t & 3) + {0, 1} of lane t / 4 (registers 4 x, 4 x + 1) and of lane t / 4 + 8.
__device__ __forceinline__ void tmem_ld_16x32(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st_16x32(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}

// This CTA's place on its lane's line of tiles, by every warp for itself: a lane sums the tiles of a run of items, the runs are added up, and the
// lane whose run has the place finds the item.  (The line has fewer than 2^31 tiles: checked by the launcher.)
__device__ __forceinline__ Plan make_plan(const AttentionArgs& a) {
    const int lane = threadIdx.x & 31;
    const int row_lane = a.lanes == 1 ? 0 : blockIdx.x % a.lanes, share = a.lanes == 1 ? blockIdx.x : blockIdx.x / a.lanes;
    const int most = a.lanes == 1 ? gridDim.x : gridDim.x / a.lanes, items = a.batch * a.blocks_per_lane;
    const int run = (items + 31) >> 5, i0 = min(lane * run, items), i1 = min(i0 + run, items);
    const int b0 = a.blocks_per_lane == 1 ? i0 : i0 / a.blocks_per_lane, rb_first = row_lane * a.blocks_per_lane;
    Piece p = {};
    int sum = 0;
    for (int i = i0, b = b0, x = i0 - b0 * a.blocks_per_lane; i < i1; ++i) {
        item_of(a, b, rb_first + x, p);
        sum += cost_of(p);
        if (++x == a.blocks_per_lane) {
            x = 0;
            ++b;
        }
    }
    int incl = sum;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, m);
        if (lane >= m) incl += o;
    }
    const int total = __shfl_sync(0xffffffffu, incl, 31);
    const int shares = max(1, min(most, (total + a.min_cost - 1) / a.min_cost));
    const int per = total / shares, rem = total - per * shares;
    const int begin = share * per + min(share, rem), end = begin + per + (share < rem);
    // the first item that begins at `begin` (items without tiles among them) or reaches beyond it
    int prefix = incl - sum, b = b0, x = i0 - b0 * a.blocks_per_lane;
    bool found = false;
    if (share < shares && i0 < i1 && prefix <= begin && incl >= begin) {
#pragma unroll 1
        for (int i = i0; i < i1; ++i) {
            item_of(a, b, rb_first + x, p);
            found = prefix == begin || prefix + cost_of(p) > begin;
            if (found) break;
            prefix += cost_of(p);
            if (++x == a.blocks_per_lane) {
                x = 0;
                ++b;
            }
        }
    }
    const unsigned hits = __ballot_sync(0xffffffffu, found);
    const int who = hits ? __ffs(hits) - 1 : 0;      // (the first lane: a later one may begin at the same place)
    Plan plan;
    plan.begin = begin; plan.end = end; plan.share = share; plan.shares = shares; plan.per = per; plan.rem = rem;
    plan.prefix = __shfl_sync(0xffffffffu, prefix, who);
    plan.b = hits ? __shfl_sync(0xffffffffu, b, who) : a.batch;      // nothing for a CTA beyond the shares
    plan.rb = __shfl_sync(0xffffffffu, rb_first + x, who);
    plan.len = __shfl_sync(0xffffffffu, p.len, who);
    plan.seen = __shfl_sync(0xffffffffu, p.seen, who);
    plan.tiles = __shfl_sync(0xffffffffu, p.tiles, who);
    return plan;
}

template <typename T>
__global__ void __launch_bounds__(kAttThreads, 1) latent_attention_kernel(const __grid_constant__ CUtensorMap map, const AttentionArgs a) {
    extern __shared__ __align__(1024) unsigned char smem[];
    AttShared& sh = *reinterpret_cast<AttShared*>(smem + kMiscOff);
    const uint32_t base = smem_u32(smem);
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    if (tid == 0) {
        for (int s = 0; s < kSlots; ++s) bar_init(&sh.slot_empty[s], 1);
        for (int s = 0; s < kTiles; ++s) {
            bar_init(&sh.kv_full[s], 1);
            bar_init(&sh.rope_empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            bar_init(&sh.p_full[s], kSoftmaxThreads);
            bar_init(&sh.pv_done[s], 1);
            bar_init(&sh.drain[s], 1);
        }
        bar_init(&sh.s_full, 1);
        bar_init(&sh.s_free, kSoftmaxThreads);
        bar_init(&sh.q_full, kSoftmaxThreads);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "n"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == 0 && elect_one()) asm volatile("prefetch.tensormap [%0];" ::"l"(&map) : "memory");
    pdl_wait_only();
    const Plan plan = make_plan(a);
    // The copying warp set the barriers up itself and need not wait for the others.
    uint32_t tmem = 0;
    if (warp == 0) {
        __syncwarp();
        asm volatile("bar.arrive 2, %0;" ::"n"(kAttThreads) : "memory");
    } else {
        tc_fence_before();
        asm volatile("bar.sync 2, %0;" ::"n"(kAttThreads) : "memory");
        tc_fence_after();
        tmem = uniform(sh.tmem);
    }
    const int rows_all = a.q_len * a.heads;
    Walk walk(a, plan, a.lanes == 1 ? 0 : (int)(blockIdx.x % a.lanes) * a.blocks_per_lane);
    Piece p = {};
    bool ok = (base & 1023) == 0;   // the swizzle is a function of the address
    // tile `it` of this CTA: its latent chunk pairs lie in ring slots 4 it .. 4 it + 3 (mod kSlots), its position values in place it mod kTiles
    int it = 0, slot = 0, place = 0;
    unsigned place_parity = 0;
    auto advance = [&] {
        ++it;
        slot += 4;
        if (slot >= kSlots) slot -= kSlots;
        if (++place == kTiles) {
            place = 0;
            place_parity ^= 1;
        }
    };
    auto slot_of = [&](int g) { return slot + g >= kSlots ? slot + g - kSlots : slot + g; };

    if (warp == 0) {
        // ── copies: the tiles of C, in boxes of box_rows rows that lie in one page ──
        const int R = a.box_rows, nb = kTileKeys / R, per_load = 32 / nb;
        unsigned wraps = 0;                        // of the slots
        while (ok && walk.next(p, false)) {
            int page_of = 0, loaded = -1;
            for (int t = p.t0; ok && t < p.t1; ++t) {
                if (loaded < 0 || t >= loaded + per_load) {   // table entries of the next 32 boxes
                    loaded = t;
                    const int key = t * kTileKeys + lane * R;
                    page_of = key < p.seen ? __ldg(a.page_table + (long long)p.b * a.table_stride + a.by_page(key)) : -1;
                }
                const int key0 = t * kTileKeys, src = min((t - loaded) * nb + lane, 31);
                const int page = __shfl_sync(0xffffffffu, page_of, src), key = key0 + lane * R;
                const bool mine = lane < nb, live = mine && key < p.seen, good = live && page >= 0 && page < a.num_pages;
                if (live && !good && a.status) atomicOr(a.status, kStatusBadPage);
                const unsigned boxes = __ballot_sync(0xffffffffu, good);
                unsigned long long m = ~0ull;
                if (boxes != (nb == 8 ? 0xffu : (1u << nb) - 1)) {
                    m = 0;
                    for (int x = 0; x < nb; ++x)
                        if (boxes >> x & 1) m |= (R == 64 ? ~0ull : (1ull << R) - 1) << (x * R);
                }
                if (p.seen - key0 < 64) m &= (1ull << (p.seen - key0)) - 1;
                const int y = key - a.by_page(key) * a.page_size, z = good ? page : a.num_pages;   // z = num_pages: outside, read as zeros
                const uint32_t row = lane * R * 128;
#pragma unroll 1
                for (int g = 0; g < 5; ++g) {
                    const int sl = slot_of(g);
                    const unsigned w = wraps + (slot + g >= kSlots);
                    uint64_t* const bar = g < 4 ? &sh.slot_empty[sl] : &sh.rope_empty[place];
                    if ((g < 4 ? w > 0 : it >= kTiles) && !bar_wait_warp(bar, g < 4 ? (w - 1) & 1 : place_parity ^ 1)) {
                        ok = false;
                        break;
                    }
                    if (g == 0) {
                        if (lane == 0) {
                            sh.mask[place] = m;
                            bar_expect(&sh.kv_full[place], kTileBytes);
                        }
                        __syncwarp();
                    }
                    if (mine) {
                        const uint32_t dst = base + row + (g < 4 ? kRingOff + sl * kSlotBytes : kRopeOff + place * kChunkBytes);
                        tma_load_3d(dst, &map, 2 * g * 64, y, z, &sh.kv_full[place]);
                        if (g < 4) tma_load_3d(dst + kChunkBytes, &map, (2 * g + 1) * 64, y, z, &sh.kv_full[place]);
                    }
                    __syncwarp();
                }
                if (slot + 4 >= kSlots) ++wraps;
                advance();
            }
        }
        // Nothing is owed to this CTA's memory when it leaves: the releases of the last tiles arrive, or, after a wait that ran out,
        // the copies in flight do (the newest tile's barrier may lack bytes that were never requested: that wait gives up).
#pragma unroll 1
        for (int s = 0; ok && s < kSlots; ++s) {
            const int uses = 4 * it / kSlots + (s < 4 * it % kSlots);
            if (uses > 0) ok = bar_wait_warp(&sh.slot_empty[s], (uses - 1) & 1);
        }
#pragma unroll 1
        for (int s = 0; s < kTiles; ++s) {
            const int uses = it / kTiles + (s < it % kTiles);
            if (uses > 0 && ok) ok = bar_wait_warp(&sh.rope_empty[s], (uses - 1) & 1);
            if (uses > 0 && !ok) bar_wait_warp(&sh.kv_full[s], (uses - 1) & 1);
        }
    } else if (warp == 1) {
        // ── S = Q . C^T ──
        int pieces = 0;
        while (ok && walk.next(p, false)) {
            ok = bar_wait_warp(&sh.q_full, pieces & 1);
            for (int t = p.t0; ok && t < p.t1; ++t) {
                ok = bar_wait_warp(&sh.kv_full[place], place_parity) && (it == 0 || bar_wait_warp(&sh.s_free, (it - 1) & 1));
                if (!ok) break;
                tc_fence_after();
                const uint32_t d = tmem + kSCol, qt = tmem + kQCol, qd = uniform(desc_k(base + kQOff));
                uint32_t cd[5];
#pragma unroll
                for (int g = 0; g < 4; ++g) cd[g] = uniform(desc_k(base + kRingOff + slot_of(g) * kSlotBytes));
                cd[4] = uniform(desc_k(base + kRopeOff + place * kChunkBytes));
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < 4 * kChunks; ++k) {
                        const int c = k >> 2;
                        const uint32_t b = cd[c >> 1] + (c & 1) * (kChunkBytes / 16) + (k & 3) * 2;
                        if (c < kQTmemChunks) umma_ts(d, qt + 8 * k, b, kIdescS<T>, k > 0);
                        else umma_ss(d, qd + (c - kQTmemChunks) * (kChunkBytes / 16) + (k & 3) * 2, b, kIdescS<T>, 1u);
                    }
                    umma_commit(&sh.s_full);
                }
                __syncwarp();
                advance();
            }
            ++pieces;
        }
        if (!ok) {   // the MMAs that were issued have to be through before the tensor memory is freed
            if (elect_one()) umma_commit(&sh.drain[0]);
            __syncwarp();
            bar_wait_warp(&sh.drain[0], 0);
        }
    } else if (warp == 2) {
        // ── O^T += C^T . P^T ──
        while (ok && walk.next(p, false)) {
            for (int t = p.t0; ok && t < p.t1; ++t) {
                ok = bar_wait_warp(&sh.kv_full[place], place_parity) && bar_wait_warp(&sh.p_full[it & 1], (unsigned)(it >> 1) & 1);
                if (!ok) break;
                tc_fence_after();
                const uint32_t pd = uniform(desc_k(base + kRopeOff + place * kChunkBytes)), acc = uniform(t > p.t0);
                uint32_t cd[4];
                int sl[4];
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    sl[g] = (int)uniform((uint32_t)slot_of(g));
                    cd[g] = uniform(desc_mn(base + kRingOff + sl[g] * kSlotBytes));
                }
                if (elect_one()) {
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) umma_ss(tmem + 64 * g, cd[g] + k * (2048 / 16), pd + k * 2, kIdescO<T>, k > 0 ? 1u : acc);
                        umma_commit(&sh.slot_empty[sl[g]]);
                    }
                    umma_commit(&sh.rope_empty[place]);
                    umma_commit(&sh.pv_done[it & 1]);
                }
                __syncwarp();
                advance();
            }
        }
        if (!ok) {
            if (elect_one()) umma_commit(&sh.drain[1]);
            __syncwarp();
            bar_wait_warp(&sh.drain[1], 0);
        }
    } else if (warp >= 4) {
        // ── Q, softmax and results ──
        // Two teams of four warps, 32 keys each; warp w of a team has rows 16 w .. (their lanes in tensor memory), a thread two rows
        // and eight keys of each.  (A thread whose wait ran out goes on to the next common barrier, where all of them leave.)
        const int team = (warp - 4) >> 2, w = warp & 3, r0 = 16 * w + (lane >> 2), r1 = r0 + 8, c0 = 32 * team + 2 * (lane & 3);
        const uint32_t quarter = (uint32_t)(32 * w) << 16;
        const int stid = tid - 128;
        // Q of a piece (behind its last row that row again: what comes of it is not stored): six chunks of its nine to tensor memory (row 16 w + i is lane 32 w + i, two
        // values per column), three to shared memory.  Its place is free: the scores of the piece before have been seen.
        // (In the order of the 16 x 256-bit store a load of the warp takes 32 bytes of eight rows; with a row per lane it touched 16 lines
        // for 16 bytes each, and Q took 6900 cycles, the table entry behind it 4700.)
        uint2 qv[3][4][2];
        auto fetch_q = [&](const Piece& n) {
            const T* q = (const T*)a.q + (long long)n.b * a.q_len * a.q_token;
            auto row_at = [&](int r) {
                const int row = min(n.rb * a.block_rows + r, rows_all - 1), j = a.by_heads(row);
                return q + j * a.q_token + (row - j * a.heads) * a.q_head;
            };
            const T *src0 = row_at(r0) + 3 * team * 64 + 4 * (lane & 3), *src1 = row_at(r1) + 3 * team * 64 + 4 * (lane & 3);
#pragma unroll
            for (int c = 0; c < 3; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    qv[c][i][0] = __ldg(reinterpret_cast<const uint2*>(src0 + c * 64 + i * 16));
                    qv[c][i][1] = __ldg(reinterpret_cast<const uint2*>(src1 + c * 64 + i * 16));
                }
            if (lane < 24) {
                const uint32_t dst = base + kQOff + (lane >> 3) * kChunkBytes + 8 * (warp - 4) * 128;
#pragma unroll
                for (int i = 0; i < 8; ++i) cp_async16(dst + i * 128 + (((lane & 7) ^ i) << 4), row_at(8 * (warp - 4) + i) + kQTmemChunks * 64 + lane * 8);
            }
        };
        auto store_q = [&] {
#pragma unroll
            for (int c = 0; c < 3; ++c) tmem_st_16x32(tmem + kQCol + 32 * (3 * team + c) + quarter, reinterpret_cast<const uint32_t*>(qv[c]));
            tmem_st_wait();
            asm volatile("cp.async.wait_all;" ::: "memory");
            proxy_fence();
            tc_fence_before();
            bar_arrive(&sh.q_full);
        };
        if (stid == 0 && !a.by_item) a.made_of[blockIdx.x] = make_int4(0, 0, 0, 0);
        // A round: the next piece's Q requested, the results of the piece before, with Q put in place half way, the next one's tiles.
        constexpr float kAhead = kLead<T> + kLazy;     // of a row's maximum before its reference
        float m0 = 0.f, m1 = 0.f, l0 = 0.f, l1 = 0.f;
        long long token0 = 0;
        Piece next;
#pragma unroll 1
        for (bool open = false; open || ok; open = true) {
            const bool more = walk.next(next, false);
            if (more) fetch_q(next);
            // The adding launch may come now.  (Earlier its blocks crowd on the SMs that have no CTA of this one, and the others stay idle.)
            else if (stid == 0) pdl_release();
            const bool whole = open && p.t0 == 0 && p.t1 == p.tiles;
            const int part = 2 * blockIdx.x + (p.t0 == 0 ? 1 : 0);
            if (open) {
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
                if (team == 0 && (lane & 3) == 0) {
                    const int row0 = p.rb * a.block_rows + r0, row1 = row0 + 8;
                    l0 += sh.team[1][r0];
                    l1 += sh.team[1][r1];
                    if (whole) {
                        sh.inv[r0] = l0 == 0.f ? 0.f : rcp(l0);
                        sh.inv[r1] = l1 == 0.f ? 0.f : rcp(l1);
                        if (a.lse) {
                            if (r0 < a.block_rows && row0 < rows_all) a.lse[token0 * a.heads + row0] = lse_of(m0, l0);
                            if (r1 < a.block_rows && row1 < rows_all) a.lse[token0 * a.heads + row1] = lse_of(m1, l1);
                        }
                    } else {
                        a.part_ml[part * kTileRows + r0] = make_float2(m0, l0);
                        a.part_ml[part * kTileRows + r1] = make_float2(m1, l1);
                    }
                }
                if (p.t0 == 0 && stid == 0 && (a.by_item || !whole)) {
                    // up to the share that holds the item's last tile
                    const int x = p.prefix + kPieceCost + p.tiles - 1, wide = plan.rem * (plan.per + 1);
                    const int last = whole ? plan.share : x < wide ? x / (plan.per + 1) : plan.rem + (x - wide) / plan.per;
                    a.made_of[a.by_item ? p.b * a.lanes * a.blocks_per_lane + p.rb : (int)blockIdx.x] = make_int4(p.b, p.rb, last - plan.share + 1, blockIdx.x);
                }
                if (whole) softmax_sync();
            }
            const int n = min(a.block_rows, rows_all - p.rb * a.block_rows), sub = lane & 3;
            // O's columns 32 x ..: rows 32 (x & 1) .. of the values 128 (x >> 1) + 32 w + lane; a team has half of them
#pragma unroll 1
            for (int y = 0; y < 4; y += a.block_rows > 32 ? 1 : 2) {
                if (y == 2 && more) store_q();
                if (!open) continue;
                const int x = 4 * team + y;
                uint32_t o[32];
                tmem_ld_32x32(tmem + 32 * x + quarter, o);
                tmem_ld_wait();
                if (whole) {
                    // a lane has one value of 32 rows; four lanes exchange theirs, so that each has four neighbouring values of eight rows
                    transpose4(o, sub);
                    int r = 32 * (x & 1) + sub;
                    T* out = (T*)a.out + token0 * a.out_token + 128 * (x >> 1) + 32 * w + (lane & ~3);
#pragma unroll
                    for (int i = 0; i < 8; ++i, r += 4) {
                        if (r < n) {
                            const int row = p.rb * a.block_rows + r, j = a.by_heads(row), h = row - j * a.heads;
                            const float f = sh.inv[r];
                            uint2 b;
                            b.x = pack2<T>(__uint_as_float(o[4 * i]) * f, __uint_as_float(o[4 * i + 1]) * f);
                            b.y = pack2<T>(__uint_as_float(o[4 * i + 2]) * f, __uint_as_float(o[4 * i + 3]) * f);
                            *reinterpret_cast<uint2*>(out + j * a.out_token + h * a.out_head) = b;
                        }
                    }
                } else {
                    // in the order in which the values lie in registers: four rows of a value are 16 bytes, a warp's 32 values 512
                    float4* out = a.part_o + (size_t)part * (kPartFloats / 4) + w * (8 * 8 * 32) + lane;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (32 * (x & 1) + 4 * i < n) out[(x * 8 + i) * 32] = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]),
                                                            __uint_as_float(o[4 * i + 3]));
                }
            }
            tc_fence_before();
            if (!more) break;
            p = next;
            token0 = (long long)p.b * a.q_len;
            if (stid == 0 && p.len > a.max_pages * a.page_size && a.status) atomicOr(a.status, kStatusBadPage);
            const int j0 = a.by_heads(p.rb * a.block_rows + r0), j1 = a.by_heads(p.rb * a.block_rows + r1);
            const int seen0 = min(p.len - a.q_len + j0 + 1, p.seen), seen1 = min(p.len - a.q_len + j1 + 1, p.seen);
            const int seen_all = min(p.len - a.q_len + a.by_heads(p.rb * a.block_rows) + 1, p.seen);    // keys that every row sees
            m0 = m1 = -INFINITY;
            l0 = l1 = 0.f;
#pragma unroll 1
            for (int t = p.t0; t < p.t1; ++t) {
                const int key0 = t * kTileKeys;
                // (waiting for O of the tile two before keeps its barrier's phases apart)
                ok = ok && (it < 2 || bar_wait(&sh.pv_done[it & 1], (unsigned)((it >> 1) - 1) & 1)) && bar_wait(&sh.kv_full[place], place_parity) &&
                     bar_wait(&sh.s_full, it & 1);
                __syncwarp();
                const unsigned long long mask = sh.mask[place];
                tc_fence_after();
                uint32_t raw[16];
                tmem_ld_16x32(tmem + kSCol + 32 * team + quarter, raw);
                tmem_ld_wait();
                tc_fence_before();
                bar_arrive(&sh.s_free);
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
                if (softmax_any(x0 > m0 + kAhead || x1 > m1 + kAhead || !ok)) {
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
                    if (x0 > m0 + kAhead) {
                        const float m = x0 - kLead<T>;
                        f0 = m0 == -INFINITY ? 1.f : ex2(m0 - m);
                        m0 = m;
                        l0 *= f0;
                    }
                    if (x1 > m1 + kAhead) {
                        const float m = x1 - kLead<T>;
                        f1 = m1 == -INFINITY ? 1.f : ex2(m1 - m);
                        m1 = m;
                        l1 *= f1;
                    }
                    if (t > p.t0) {
                        if (team == 0 && (lane & 3) == 0) {
                            sh.factor[r0] = f0;
                            sh.factor[r1] = f1;
                        }
                        softmax_sync();
                        ok = bar_wait(&sh.pv_done[(it - 1) & 1], (unsigned)((it - 1) >> 1) & 1);
                        __syncwarp();
                        tc_fence_after();
#pragma unroll 1
                        for (int x = 4 * team; x < 4 * team + 4; x += a.block_rows > 32 ? 1 : 2) {
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
                unsigned char* pr = smem + kRopeOff + place * kChunkBytes + 4 * (lane & 3);
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
#pragma unroll 1
                    for (int c = 0; c < 8; ++c)
#pragma unroll 1
                        for (int i = stid; i < n; i += kSoftmaxThreads)
                            *reinterpret_cast<uint4*>(smem + kRingOff + slot_of(c >> 1) * kSlotBytes + (c & 1) * kChunkBytes + first * 128 + i * 16) =
                                make_uint4(0, 0, 0, 0);
                }
                proxy_fence();
                tc_fence_before();
                bar_arrive(&sh.p_full[it & 1]);
                advance();
            }
        }
        // Items of this CTA that have no tiles: no row of theirs sees a key.
        Walk none(a, plan, walk.rb0);
        while (ok && none.next(p, true)) {
            const int n = min(a.block_rows, rows_all - p.rb * a.block_rows);
            if (stid == 0 && a.by_item) a.made_of[p.b * a.lanes * a.blocks_per_lane + p.rb] = make_int4(0, 0, 0, 0);
            for (int r = warp - 4; r < n; r += 8) {
                const int row = p.rb * a.block_rows + r, j = a.by_heads(row), h = row - j * a.heads;
                const long long token = (long long)p.b * a.q_len + j;
                uint4* o = reinterpret_cast<uint4*>((T*)a.out + token * a.out_token + h * a.out_head);
                o[lane] = o[lane + 32] = make_uint4(0, 0, 0, 0);
                if (lane == 0 && a.lse) a.lse[token * a.heads + h] = -INFINITY;
            }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (!ok && lane == 0 && a.status) atomicOr(a.status, kStatusTimeout);
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kTmemCols) : "memory");
    }
}

// Adds up the parts of the row blocks that several CTAs shared.  The parts lie in the second place of the CTA that begins the block and in
// the first places of the CTAs after it in its lane.  A unit of work is four rows and 32 of every 128 values (of all four 128s, or of one).  One warp adds up to four parts of a unit; of more parts `team` warps take every team-th each and meet in shared memory.
// How large a team, and with it the grid, the launcher chooses by the number of row blocks: a few may have up to 148 parts each,
// many have about two, and then the blocks beyond the first return at once.
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int y = 16; y; y >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, y));
    return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int y = 16; y; y >>= 1) v += __shfl_xor_sync(0xffffffffu, v, y);
    return v;
}

constexpr int kCombineThreads = 256, kCombineWarps = kCombineThreads / 32, kCombineAlone = 4;

template <typename T, int GN>
__global__ void __launch_bounds__(kCombineThreads, 2) latent_combine_kernel(const AttentionArgs a, int most) {
    constexpr int kSplit = 4 / GN, kDepth = 8 / GN;     // parts whose loads are in flight together
    __shared__ float4 sums[kCombineWarps][GN][32];
    __shared__ float4 weights[kCombineWarps][kCombineAlone > kMaxGrid / kCombineWarps ? kCombineAlone : (kMaxGrid + kCombineWarps - 1) / kCombineWarps];
    __shared__ float4 tops[2 * kCombineWarps];
    pdl_enter();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rows_all = a.q_len * a.heads;
    const int4 own = a.made_of[blockIdx.x];      // (row blocks first: the blocks that return at once come last)
    const int parts = own.z, c = own.w, team = parts <= kCombineAlone ? 1 : most;
    const int x = blockIdx.y * kCombineWarps + warp, mate = x & (team - 1), unit = x / team;
    if (parts < 2 || unit >= a.block_rows * kSplit) return;      // (the same for all warps of a block: team divides their number)
    // (an entry that no CTA has written, after a wait that ran out, is whatever the workspace held)
    if (c < 0 || parts > kMaxGrid || c + (parts - 1) * a.lanes >= kMaxGrid || own.x < 0 || own.x >= a.batch || own.y < 0 || own.y >= a.lanes * a.blocks_per_lane)
        return;
    const int u = unit / kSplit;
    // rows r .. r + 3 of the block, values 128 g + 32 w + lane with g in [g0, g0 + GN)
    const int w = u & 3, r = (u >> 2) * 4, g0 = GN * (unit % kSplit), row0 = own.y * a.block_rows + r;
    if (row0 >= rows_all) return;              // (a block whose warps meet has one group of rows)
    auto place = [&](int k) { return 2 * (c + k * a.lanes) + (k == 0); };
    const float4* src = a.part_o + (w * 64 + (2 * g0 + (r >> 5)) * 8 + ((r & 31) >> 2)) * 32 + lane;
    const float4* ml = reinterpret_cast<const float4*>(a.part_ml + r);     // (m, l) of two rows each
    constexpr int kMl = kTileRows / 2;
    float4 v[kDepth][GN];
    auto fetch = [&](int k) {
#pragma unroll
        for (int i = 0; i < kDepth; ++i)
#pragma unroll
            for (int g = 0; g < GN; ++g) v[i][g] = src[(size_t)place(min(k + i * team, parts - 1)) * (kPartFloats / 4) + g * (2 * 8 * 32)];
    };
    fetch(mate);
    // The rows' largest reference, the parts' weights relative to it, the sums.  A warp alone does it for itself; a team's block, which has one
    // group of rows, does it once, a part per thread (every warp for itself: 2000 warps asked for the same lines, 8 us).
    float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
    float4 l = make_float4(0.f, 0.f, 0.f, 0.f), p, q;
    p.x = p.z = q.x = q.z = -INFINITY;
    p.y = p.w = q.y = q.w = 0.f;
    const int mine = team > 1 ? (int)threadIdx.x : lane;
    if (mine < parts) {
        p = ml[place(mine) * kMl];
        q = ml[place(mine) * kMl + 1];
    }
    m0 = warp_max(p.x); m1 = warp_max(p.z); m2 = warp_max(q.x); m3 = warp_max(q.z);
    if (team > 1) {
        if (lane == 0) tops[warp] = make_float4(m0, m1, m2, m3);
        __syncthreads();
#pragma unroll 1
        for (int y = 0; y < (kMaxGrid + 31) / 32; ++y) {
            const float4 t = tops[y];
            m0 = fmaxf(m0, t.x); m1 = fmaxf(m1, t.y); m2 = fmaxf(m2, t.z); m3 = fmaxf(m3, t.w);
        }
    }
    const float4 f = make_float4(weight_of(p.x, m0), weight_of(p.z, m1), weight_of(q.x, m2), weight_of(q.z, m3));
    l = make_float4(warp_sum(f.x * p.y), warp_sum(f.y * p.w), warp_sum(f.z * q.y), warp_sum(f.w * q.w));
    float4* const weight = team > 1 ? weights[0] : weights[warp];
    if (mine < parts) weight[mine] = f;
    if (team > 1) {
        if (lane == 0) tops[kCombineWarps + warp] = l;
        __syncthreads();
        l = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int y = 0; y < (kMaxGrid + 31) / 32; ++y) {
            const float4 t = tops[kCombineWarps + y];
            l.x += t.x; l.y += t.y; l.z += t.z; l.w += t.w;
        }
    } else {
        __syncwarp();
    }
    float4 o[GN];
#pragma unroll
    for (int g = 0; g < GN; ++g) o[g] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int k = mate; k < parts; k += kDepth * team) {
        if (k != mate) fetch(k);
#pragma unroll
        for (int i = 0; i < kDepth; ++i) {
            const int ki = k + i * team;
            if (ki < parts) {
                const float4 x = weight[ki];
#pragma unroll
                for (int g = 0; g < GN; ++g) {
                    o[g].x = fmaf(x.x, v[i][g].x, o[g].x); o[g].y = fmaf(x.y, v[i][g].y, o[g].y);
                    o[g].z = fmaf(x.z, v[i][g].z, o[g].z); o[g].w = fmaf(x.w, v[i][g].w, o[g].w);
                }
            }
        }
    }
    if (team > 1) {
#pragma unroll
        for (int g = 0; g < GN; ++g) sums[warp][g][lane] = o[g];
        __syncthreads();
        if (mate > 0) return;
#pragma unroll 1
        for (int y = 1; y < team; ++y) {
#pragma unroll
            for (int g = 0; g < GN; ++g) {
                const float4 s = sums[warp + y][g][lane];
                o[g].x += s.x; o[g].y += s.y; o[g].z += s.z; o[g].w += s.w;
            }
        }
    }
    auto store = [&](int e, float m, float sum, auto value) {
        const int row = row0 + e;
        if (row >= rows_all) return;
        const int j = a.by_heads(row), h = row - j * a.heads;
        const long long token = (long long)own.x * a.q_len + j;
        const float inv = sum == 0.f ? 0.f : rcp(sum);
        T* out = (T*)a.out + token * a.out_token + h * a.out_head + 128 * g0 + 32 * w + lane;
#pragma unroll
        for (int g = 0; g < GN; ++g) out[128 * g] = from_float<T>(value(o[g]) * inv);
        if (w == 0 && g0 == 0 && lane == 0 && a.lse) a.lse[token * a.heads + h] = lse_of(m, sum);
    };
    store(0, m0, l.x, [](const float4& f) { return f.x; });
    store(1, m1, l.y, [](const float4& f) { return f.y; });
    store(2, m2, l.z, [](const float4& f) { return f.z; });
    store(3, m3, l.w, [](const float4& f) { return f.w; });
}

namespace {

FastDiv fast_div(unsigned d, int bits) {
    int log = 0;
    while ((1u << log) < d) ++log;
    const int shift = bits + log;
    return FastDiv{(unsigned)(((1ull << shift) + d - 1) / d), (unsigned)shift};
}

constexpr size_t kMadeBytes = kMaxGrid * sizeof(int4), kMlBytes = 2 * (size_t)kMaxGrid * kTileRows * sizeof(float2);
constexpr size_t kAttWorkspace = kMadeBytes + kMlBytes + 2 * (size_t)kMaxGrid * kPartFloats * sizeof(float);

template <typename T>
int launch_attention(const CUtensorMap& map, const AttentionArgs& a, int grid, cudaStream_t st) {
    int r = allow_smem<latent_attention_kernel<T>>(kAttSmem);
    if (r) return r;
    r = launch_latent(latent_attention_kernel<T>, dim3((unsigned)grid), kAttThreads, kAttSmem, st, map, a);
    if (r) return r;
    const long long items = (long long)a.batch * a.lanes * a.blocks_per_lane;
    const int made = a.by_item ? (int)items : grid;
    // As many warps for a part's bytes as about two blocks per SM have: more blocks come in waves (four row blocks in 1024 blocks: 12 us
    // instead of 5).
    const int room = 2 * sm_count() + 24, units = a.block_rows / kCombineWarps * made;
    const int split = units * 32 <= room ? 4 : 1, team = units * 8 <= room ? 8 : units * 4 <= room ? 4 : 2;
    const dim3 blocks((unsigned)made, (unsigned)(a.block_rows * team * split / kCombineWarps));
    return split == 4 ? launch_latent(latent_combine_kernel<T, 1>, blocks, kCombineThreads, 0, st, a, team)
                      : launch_latent(latent_combine_kernel<T, 4>, blocks, kCombineThreads, 0, st, a, team);
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
    // (without rows or sequences the address of an empty tensor is null)
    if ((batch != 0 && (!page_table || !seq_lens || (q_len != 0 && (!q || !out)))) || !cache || !workspace) return VIB3_ERR_NULL;
    if (dtype != L_F16 && dtype != L_BF16) return VIB3_ERR_UNSUPPORTED;
    if (page_size % 8) return VIB3_ERR_UNSUPPORTED;
    // (the copying warp looks up table entries for 32 boxes at once, up to 2048 keys beyond the length, and key numbers have 32 bits)
    if (batch < 0 || q_len < 0 || heads <= 0 || heads > kLatentMaxHeads || num_pages <= 0 || num_pages > 0x7fffffff || page_size <= 0 ||
        page_size > (1 << 20) || max_pages_per_seq <= 0 || (long long)max_pages_per_seq * page_size > 0x7ffff000 ||
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

    AttentionArgs a;
    a.q = q; a.q_token = q_token_stride; a.q_head = q_head_stride;
    a.page_size = page_size; a.num_pages = (int)num_pages;
    a.box_rows = page_size % 64 == 0 ? 64 : page_size % 32 == 0 ? 32 : page_size % 16 == 0 ? 16 : 8;
    a.page_table = page_table; a.table_stride = table_stride; a.max_pages = max_pages_per_seq;
    a.seq_lens = seq_lens; a.batch = batch; a.q_len = q_len; a.heads = heads;
    a.by_heads = fast_div((unsigned)heads, 27);
    a.by_page = fast_div((unsigned)page_size, 31);
    a.scale_log2 = scale * 1.4426950408889634074f;
    a.out = out; a.out_token = out_token_stride; a.out_head = out_head_stride;
    a.lse = lse_or_null; a.status = status;
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    a.made_of = reinterpret_cast<int4*>(ws);
    a.part_ml = reinterpret_cast<float2*>(ws + kMadeBytes);
    a.part_o = reinterpret_cast<float4*>(ws + kMadeBytes + kMlBytes);
    const int sms = sm_count() < kMaxGrid ? sm_count() : kMaxGrid;
    const long long rows = (long long)q_len * heads, most_tiles = ((long long)max_pages_per_seq * page_size + kTileKeys - 1) / kTileKeys;
    // Half row blocks where the whole ones would leave half of the SMs without work: the cache is then read twice (from L2), the
    // results of a CTA, 128 KB at 27 bytes per cycle, are halved.
    a.block_rows = rows <= 32 || (rows + kTileRows - 1) / kTileRows * batch * most_tiles <= sms ? kTileRows / 2 : kTileRows;
    const int blocks = (int)((rows + a.block_rows - 1) / a.block_rows);
    a.lanes = blocks <= 8 ? blocks : 1;
    a.blocks_per_lane = blocks / a.lanes;
    // the kernel counts tiles (and what a row block costs beside them) in 32 bits
    if ((long long)batch * a.blocks_per_lane * (most_tiles + kPieceCost) > 0x7fffff00) return VIB3_ERR_COUNT;
    a.by_item = (long long)batch * blocks <= kMaxGrid;
    a.min_cost = kMinCost;
    const int grid = sms / a.lanes * a.lanes;

    if (!tensor_map_encoder()) return VIB3_ERR_UNSUPPORTED;
    CUtensorMap map;
    if (!map_3d(&map, dtype, cache, kLatentRow, page_size, num_pages, row_stride, page_stride, a.box_rows, 1))
        return VIB3_ERR_SHAPE;
    return dtype == L_F16 ? launch_attention<__half>(map, a, grid, (cudaStream_t)stream)
                          : launch_attention<__nv_bfloat16>(map, a, grid, (cudaStream_t)stream);
}
