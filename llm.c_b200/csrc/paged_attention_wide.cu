// Attention over a key / value cache in pages where a cached head has many query rows: prompts, parts of prompts behind a context, trees of drafted tokens.
//
// A row tile holds 128 rows of ONE cached head: 128 / G tokens with the G query heads of each, so that grouped heads share every key and value that is loaded.  A piece of work is a pair
// of adjacent row tiles (slots A and B) with the keys that the later one sees, in units of 128 keys; blocks have equal shares of all units (paged.cuh), so that prompts of any lengths, and a
// few drafted tokens over a long cache, fill the SMs alike.
//
// Per block: a warp that lists the pieces (it finds the block's share while the others set up barriers and tensor memory), a TMA warp, an issuer, a warp that cleans values, and four softmax warps to each slot.
//   * K and V tiles arrive page by page: the boxes of a tile (a page each, or 128 rows of a larger one) are issued by as many lanes, each of which looks its page up in the table one tile
//     ahead.  A box behind the sequence's last page, or of a page that the table names wrongly, lies outside the tensor map and arrives as zeros.
//   * Slots of the last page behind the sequence's length may hold anything.  Scores there are replaced, not added to; but a probability of zero times a value that is not finite is not
//     zero, so the cleaning warp overwrites these rows of the last V tile with zeros before the product reads it.
//   * S = Q K^T of a slot goes to tensor memory, one thread owns a row of 128 scores, P goes back as bf16 over the scores, in two halves, and is the A operand of O += P V, which begins
//     with the first half (16 trees of 64 tokens over up to 4096 keys 57.5 us, P in one piece 62; prompts the same).  The slots alternate: one's products run under the other's
//     exponentials.  Rounding P to bf16 adds an error of the size of the output's own rounding (0.0019 to 0.0022 of the result's norm from 64 bits, 0.0016 with 16 bits of P, which would take a
//     second product of the same length); the sums l are of the probabilities before it, in fp32.
//   * O stays in tensor memory.  It is rescaled when the maximum of a row of the warp has grown by 8 (base 2) over the one that its probabilities refer to; until then they are as large as
//     2^8, which fp32 sums and bf16 roundings do not mind.  A prompt of 8192 tokens, 32 heads on 8 of 128, takes 482 to 510 us.  (When they came, the lazy rescaling and arithmetic in pairs took 50 us
//     off it, the registers that the other warps do not need given to the softmax warps 27 more.)
//   * Tried and slower, the same prompt: an eighth of the exponentials as polynomials 492 instead of 482 us, a quarter 509, half 550; a tile's maxima taken beside its exponentials, relative to the
//     maximum so far, 496; before the steps above, tiles in two halves of 64 keys with room for both halves' scores 744 instead of 587 (products of 64 columns, and twice as many turns); slot B
//     started half a tile late, the same.
//   * A piece that lies in one share is divided by l and stored; parts of a piece go to the workspace in fp32, channel by channel so that a warp's stores are whole lines.
//
// TMEM columns: S_A [0,128)  S_B [128,256)  O_A [256,384)  O_B [384,512);  P_X: the first 64 columns of S_X (128 bf16 per row)
#include "paged_attention_ops.h"
#include "pdl.cuh"

namespace {

constexpr int BT = 128;
constexpr int CHUNK_BYTES = BT * 64 * 2;            // 16 KB: 128 rows x 64 channels, 128-byte swizzled
constexpr int TILE_BYTES = 2 * CHUNK_BYTES;
constexpr int RING = 5;                             // K_0 V_0 K_1 V_1 ... tiles in flight
constexpr int QUEUE = 4;                            // pieces listed ahead
constexpr int THREADS = 384;
constexpr int REGS_LOW = 104, REGS_HIGH = 200;      // of the 168 a thread that the block is launched with
static_assert(128 * REGS_LOW + 256 * REGS_HIGH <= THREADS * 168, "registers of the block");
constexpr int TMEM_COLS = 512;
constexpr int P_FIRST = 64;                         // probabilities of a tile that go back first
constexpr int SMEM = 2 * TILE_BYTES + RING * TILE_BYTES + 1024;                     // Q tiles, K / V ring, barriers and queue
static_assert(SMEM <= 232448, "shared memory of one block");

struct WideArgs {
    PagedAttention p;
    int G, tokens;        // query heads of a cached one; tokens of a row tile: 128 / G
    FastDiv by_step;      // two row tiles' tokens
    int ks;               // 16-channel steps of the head
    int over;             // units that a piece counts besides its keys: what it takes to begin and to end one
    // the first p pairs of a prompt need the sum of ceil(i step / 128) key tiles of new tokens, i = 1 .. p: new_tiles[p] up to a period of 2^period_log2 pairs, in which a pair's rises by `rise`
    int period_log2, rise;
    unsigned short new_tiles[BT + 1];
    int box;              // rows of a page that one copy brings
    float scale_log2e;
};

// The pieces of one sequence, for one cached head
struct WidePieces {
    PagedSpan s;
    int step;             // tokens of a pair of row tiles
    int pairs, over;
    int context;          // key tiles that the cached context takes
    const unsigned short* new_tiles;
    bool causal;          // pairs see as many keys as their last token; otherwise (trees, sequences with fewer keys than new tokens) all
    DEVINL void of(const WideArgs& a, const unsigned short* new_tiles_, const PagedSpan& span) {
        s = span;
        new_tiles = new_tiles_;
        step = 2 * a.tokens;
        over = a.over;
        pairs = a.by_step(s.count + step - 1);
        causal = !a.p.tree && s.count <= s.keys;
        context = (s.keys - s.count + BT - 1) / BT;
    }
    DEVINL int all() const { return s.keys > 0 ? (s.keys + BT - 1) / BT : 1; }
    DEVINL int tiles(int p) const { return causal && p + 1 < pairs ? (s.keys - s.count + (p + 1) * step + BT - 1) / BT : all(); }
    // Units of a pair: `over`, its key tiles, and where context and new tokens together need one tile less than each by itself that one, so that the units in front of a pair are known
    // without adding them up.  The keys are the last of them.
    DEVINL int lead(int p) const { return over + (causal && p + 1 < pairs ? context + ((p + 1) * step + BT - 1) / BT - tiles(p) : 0); }
    // Units of the pairs in front of p.  (Nothing here passes 2^30: a causal sequence of n pairs has n step keys or more, and the host, which counts every pair with all keys that the table has room
    // for, lets n^2 step / 128 < 2^30 through; q is n where step is 128 or 256, and n by at least 128 / step where it is less.)
    DEVINL int in_front(const WideArgs& a, int p) const {
        if (!causal) return p * (over + all());
        const int n = min(p, pairs - 1), q = n >> a.period_log2, r = n & ((1 << a.period_log2) - 1);       // (the last pair sees all keys)
        return (p > n ? over + all() : 0) + n * (over + context) + a.rise * ((q * (q - 1) / 2 << a.period_log2) + r * q) + q * new_tiles[1 << a.period_log2] + new_tiles[r];
    }
    DEVINL int units(const WideArgs& a) const { return pairs ? in_front(a, pairs) : 0; }
    // The last pair with no more than `off` units in front of it; a warp tries 32 at a time
    DEVINL int pair_of(const WideArgs& a, int off) const {
        int lo = 0, n = pairs;
        while (n > 1) {
            const int gap = (n + 31) / 32, at = lo + (threadIdx.x & 31) * gap;
            const int under = __popc(__ballot_sync(0xffffffffu, at < lo + n && in_front(a, at) <= off)) - 1;
            n = min(gap, n - under * gap);
            lo += under * gap;
        }
        return lo;
    }
};

// What the roles of a block are told about a piece, or about the part of it that lies in the block's share
struct WideItem {
    int n;                // key tiles; 0: no more pieces
    int j0;               // the first of them
    int b, g, first, count, keys, token;      // token: the first of slot A
    int has_b;
    int whole;            // all keys: the result is stored; otherwise a partial, number `part` of the workspace
    int part;
    int clean;            // the last tile has slots behind the sequence's length
};

// The workspace: what is to be joined, for each block; two partials for each block, of 8 groups of 32 rows, each channel by channel and then the maxima (base 2) and the sums
DEVINL float* wide_part(float* ws, int blocks, int hs, int part, int group) {
    return ws + blocks * (sizeof(PagedJoin) / 4) + ((size_t)part * 8 + group) * (32 * (hs + 2));
}

__global__ void __launch_bounds__(THREADS, 1)
paged_wide_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const PagedCache c, const __grid_constant__ WideArgs a) {
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* sQ = smem;                                   // [A, B]
    uint8_t* sKV = sQ + 2 * TILE_BYTES;                   // [RING]
    uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + RING * TILE_BYTES);
    uint64_t* q_full = bars + 0;      // [2 slots]
    uint64_t* q_empty = bars + 2;     // [2] the slot's last S of the piece is complete         (1 commit)
    uint64_t* kv_full = bars + 4;     // [RING]
    uint64_t* kv_empty = bars + 9;    // [RING]
    uint64_t* s_full = bars + 14;     // [2] S_X(t) complete, and with it every earlier product (1 commit)
    uint64_t* p_ready = bars + 16;    // [2] P_X(t) is in TMEM (and O_X rescaled if needed)     (4 arrivals)
    uint64_t* o_full = bars + 18;     // [2] the piece's O_X is complete                        (1 commit)
    uint64_t* o_free = bars + 20;     // [2] the slot's warps have read O_X                     (4 arrivals)
    uint64_t* v_here = bars + 22;     // a V tile with slots behind the length has arrived      (the issuer)
    uint64_t* v_clean = bars + 23;    // it has zeros there                                     (the cleaning warp)
    uint64_t* item_full = bars + 24;  // [QUEUE]
    uint64_t* item_empty = bars + 28; // [QUEUE] (11 warps)
    uint64_t* p_rest = bars + 32;     // [2] the rest of P_X(t)                                 (4 arrivals)
    WideItem* queue = reinterpret_cast<WideItem*>(bars + 46);     // [QUEUE]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(queue + QUEUE);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    unsigned short* new_tiles = reinterpret_cast<unsigned short*>(tmem_slot + 2);        // [129]
    static_assert(46 * 8 + QUEUE * sizeof(WideItem) + 8 + (BT + 1) * 2 <= 1024, "barriers, queue, key tiles of new tokens");

    const int warp = warp_index(), lane = threadIdx.x & 31;
    unsigned int* status = a.p.status;
    if (threadIdx.x == 0) {
        if ((smem_u32(smem) & 1023u) != 0) record_error(status, ST_BAD_ARG, 0x4C);
        for (int i = 0; i < 2; i++) {
            mbar_init(&q_full[i], 1); mbar_init(&q_empty[i], 1);
            mbar_init(&s_full[i], 1); mbar_init(&p_ready[i], 4); mbar_init(&p_rest[i], 4); mbar_init(&o_full[i], 1); mbar_init(&o_free[i], 4);
        }
        for (int i = 0; i < RING; i++) { mbar_init(&kv_full[i], 1); mbar_init(&kv_empty[i], 1); }
        for (int i = 0; i < QUEUE; i++) { mbar_init(&item_full[i], 1); mbar_init(&item_empty[i], 11); }
        mbar_init(v_here, 1); mbar_init(v_clean, 1);
        *abort_flag = 0;
        mbar_fence_init();
        tma_prefetch_desc(&tmQ); tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV);
    }
    if (warp == 1) { tmem_alloc(tmem_slot, TMEM_COLS); tmem_relinquish(); }
    if (warp == 3) {
        for (int i = lane; i <= 1 << a.period_log2; i += 32) new_tiles[i] = a.new_tiles[i];
        __syncwarp();
    }
    pdl_wait();
    pdl_trigger();
    // the lister finds the block's share while the others set up
    PagedPlace place = {};
    int total = 0;
    if (warp == 3)
        total = paged_find(c, a.p.N, status, 0x4B, [&](const PagedSpan& span) { WidePieces w; w.of(a, new_tiles, span); return w.units(a) * c.heads; }, [&](int sum) {
            const PagedShares sh(sum, gridDim.x);
            return (int)blockIdx.x < sh.blocks ? sh.first(blockIdx.x) : -1;
        }, place);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int nch = c.hs > 64 ? 2 : 1;

    // the roles read the queue in order; a warp gives an entry back when it needs it no longer
    auto take = [&](uint32_t i, WideItem& it) {
        if (!__all_sync(0xffffffffu, mbar_wait_relaxed(&item_full[i % QUEUE], (i / QUEUE) & 1, abort_flag, status, 0x530))) { it.n = 0; return false; }
        it = queue[i % QUEUE];
        return it.n > 0;
    };
    auto give_back = [&](uint32_t i) { __syncwarp(); if (lane == 0) mbar_arrive(&item_empty[i % QUEUE]); };

    // 128 x REGS_LOW + 256 x REGS_HIGH registers: what the block was launched with
    if (warp < 4) {
    regs_shrink<REGS_LOW>();
    if (warp == 3) {
        // ---------------------------------------------------------------- lists the pieces
        const PagedShares shares(total, gridDim.x);
        const bool works = (int)blockIdx.x < shares.blocks;
        const int first = works ? shares.first(blockIdx.x) : 0;
        int end = works ? shares.first(blockIdx.x + 1) : 0;
        WidePieces w = {};
        int g = 0, p = 0, off = 0;
        if (end > first) w.of(a, new_tiles, place.s);
        if (w.pairs == 0) end = first;
        if (end > first) {
            const int per_head = w.units(a);
            g = place.offset / per_head;
            off = place.offset - g * per_head;
            p = w.pair_of(a, off);
        }
        if (lane == 0) {
            uint32_t i = 0;
            bool ok = true;
            auto put = [&](const WideItem& it) {
                ok = ok && mbar_wait_relaxed(&item_empty[i % QUEUE], ((i / QUEUE) & 1) ^ 1, abort_flag, status, 0x531);
                if (ok) { queue[i % QUEUE] = it; mbar_arrive(&item_full[i % QUEUE]); }
                i++;
            };
            int left = end - first;
            const WidePieces begun = w;
            const int g0 = g, p0 = p, x0 = off - w.in_front(a, p) - w.lead(p);         // the first unit of keys; below 0: the share begins in front of them
            if (left > 0) {
                int b = place.b;
                int x = x0;
                while (left > 0 && ok) {
                    const int tiles = w.tiles(p), j0 = max(0, x), n = min(tiles, x + left) - j0;
                    left -= min(tiles, x + left) - x;
                    if (n > 0) {
                        WideItem it;
                        it.n = n; it.j0 = j0; it.b = b; it.g = g; it.first = w.s.first; it.count = w.s.count; it.keys = w.s.keys; it.token = p * w.step;
                        it.has_b = it.token + a.tokens < w.s.count;
                        it.whole = n == tiles;
                        it.part = 2 * blockIdx.x + (j0 == 0);
                        it.clean = (j0 + n) * BT > w.s.keys;
                        put(it);
                        if (a.p.tree && w.s.count > 64) record_error(status, ST_BAD_ARG, 0x49);
                    }
                    if (++p == w.pairs) {
                        p = 0;
                        if (++g == c.heads && left > 0) {
                            g = 0;
                            do {
                                if (++b >= c.sequences) { left = 0; break; }
                                w.of(a, new_tiles, paged_span(c, b, a.p.N, status, 0x4B));
                            } while (w.pairs == 0);
                        }
                    }
                    x = -w.lead(p);
                }
            }
            WideItem none;
            none.n = 0;
            put(none);
            // whether this is the first share that begins inside the piece, for the kernel that joins the parts
            PagedJoin join = {0, begun.s.first, begun.s.count, g0, p0 * begun.step};
            if (works && x0 > 0) {
                const int tile0 = first - x0;                     // where the first of the piece's keys lies among all units
                if (shares.share_of(tile0) == (int)blockIdx.x - 1) join.parts = shares.share_of(tile0 + begun.tiles(p0) - 1) - (int)blockIdx.x + 2;
            }
            reinterpret_cast<PagedJoin*>(a.p.ws)[blockIdx.x] = join;
        }
    } else if (warp == 0) {
        // ---------------------------------------------------------------- TMA producer: a lane for each box of a tile
        const int boxes = BT / a.box, lanes = boxes * nch;
        const int mine = lane % boxes, chunk = lane / boxes;
        const bool issues = lane < lanes;
        uint32_t n = 0, nx[2] = {0, 0};        // ring tiles, pieces of each slot so far
        WideItem it;
        bool ok = true;
        for (uint32_t i = 0; ok && take(i, it); i++) {
            // the table's entry for a box, and the page: one behind the last where the box lies behind the sequence or the table names none
            auto entry_of = [&](int j) {
                const int slot = j * BT + mine * a.box;
                return issues && slot < it.keys ? c.table[it.b * c.table_row + (slot >> c.page_shift)] : c.pages;
            };
            auto page_of = [&](int entry, int j) {
                if ((unsigned)entry < (unsigned)c.pages) return entry;
                if (issues && j * BT + mine * a.box < it.keys) record_error(status, ST_BAD_ARG, 0x4D);
                return c.pages;
            };
            int entry = entry_of(it.j0);
            const int rows = a.G * a.tokens;
            for (int x = 0; x < (it.has_b ? 2 : 1) && ok; x++) {
                ok = __all_sync(0xffffffffu, mbar_wait_relaxed(&q_empty[x], (nx[x] & 1) ^ 1, abort_flag, status, 0x502)) != 0;
                if (!ok) break;
                nx[x]++;
                if (lane == 0) {
                    mbar_expect_tx(&q_full[x], nch * rows * 128);
                    for (int ch = 0; ch < nch; ch++)
                        tma_load_3d(sQ + x * TILE_BYTES + ch * CHUNK_BYTES, &tmQ, &q_full[x], ch * 64, it.g * a.G, it.first + it.token + x * a.tokens);
                }
                __syncwarp();
            }
            for (int j = it.j0; j < it.j0 + it.n && ok; j++) {
                const int page = page_of(entry, j);
                if (j + 1 < it.j0 + it.n) entry = entry_of(j + 1);
                const int row = (j * BT + mine * a.box) & ((1 << c.page_shift) - 1);
                for (int kv = 0; kv < 2 && ok; kv++, n++) {
                    const uint32_t st = n % RING;
                    ok = __all_sync(0xffffffffu, mbar_wait_relaxed(&kv_empty[st], ((n / RING) & 1) ^ 1, abort_flag, status, 0x500)) != 0;
                    if (!ok) break;
                    if (lane == 0) mbar_expect_tx(&kv_full[st], nch * CHUNK_BYTES);
                    __syncwarp();
                    if (issues) tma_load_4d(sKV + st * TILE_BYTES + chunk * CHUNK_BYTES + mine * a.box * 128, kv ? &tmV : &tmK, &kv_full[st], chunk * 64, it.g, row, page);
                    __syncwarp();
                }
            }
            give_back(i);
        }
    } else if (warp == 2) {
        // ---------------------------------------------------------------- zeros behind the length in the last V tile of a sequence
        // (told by the issuer, which follows the ring: this warp would not know one round of the ring from the next but one)
        uint32_t kabs = 0, cleaned = 0;
        WideItem it;
        bool ok = true;
        for (uint32_t i = 0; ok && take(i, it); i++) {
            if (it.clean) {
                const uint32_t pos = 2 * (kabs + it.n - 1) + 1;
                ok = mbar_wait_relaxed(v_here, cleaned++ & 1, abort_flag, status, 0x532) && mbar_wait_relaxed(&kv_full[pos % RING], (pos / RING) & 1, abort_flag, status, 0x534);
                ok = __all_sync(0xffffffffu, ok) != 0;
                if (ok) {
                    uint8_t* v = sKV + (pos % RING) * TILE_BYTES;
                    const int from = max(0, it.keys - (it.j0 + it.n - 1) * BT);
                    for (int k = from * 8 + lane; k < BT * 8; k += 32)
                        for (int ch = 0; ch < nch; ch++) *reinterpret_cast<uint4*>(v + ch * CHUNK_BYTES + k * 16) = make_uint4(0, 0, 0, 0);
                    fence_async_smem();
                }
                __syncwarp();
                if (lane == 0 && ok) mbar_arrive(v_clean);
            }
            kabs += it.n;
            give_back(i);
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- issuer: per piece  S_A(0) S_B(0), then for every key tile j
        // O_A += P_A(j) V_j, S_A(j+1), O_B += P_B(j) V_j, S_B(j+1); slot B's last step has the next piece's S_A(0) in front of it
        const bool leader = elect_one();
#define WAIT_ALL(bar, parity, code) (__all_sync(0xffffffffu, mbar_wait_relaxed(bar, parity, abort_flag, status, code)) != 0)
        constexpr uint32_t idesc_s = umma_idesc_bf16(BT, BT, 0, 0);                             // Q (K-major) x K (K-major)
        const uint32_t idesc_o = umma_idesc_bf16(BT, 0, 0, 1) | ((uint32_t)(a.ks * 2) << 17);   // P (TMEM) x V (N-major), N = 16 ks
        constexpr uint32_t TILE_UNITS = TILE_BYTES / 16, CHUNK_UNITS = CHUNK_BYTES / 16;
        const uint64_t dQ0 = umma_desc_sw128(smem_u32(sQ), 16, 1024), dK0 = umma_desc_sw128(smem_u32(sKV), 16, 1024);
        const uint64_t dV0 = umma_desc_sw128(smem_u32(sKV), CHUNK_BYTES, 1024);
        const int ks = a.ks;
        uint32_t tp[2] = {0, 0};          // P V products issued per slot
        uint32_t qn[2] = {0, 0};          // Q tiles (pieces) whose first S has been issued per slot
        uint32_t on[2] = {0, 0};          // pieces whose first P V has been issued per slot
        uint32_t kabs = 0;                // key tiles of earlier pieces: K_j sits at ring position 2 (kabs + j), V_j behind it
        uint32_t cleaned = 0;
        auto kv_wait = [&](uint32_t pos, uint32_t code) { return WAIT_ALL(&kv_full[pos % RING], (pos / RING) & 1, code); };
        // S_x of the key tile at ring position pos; first: the slot's Q tile is new; the slot that reads a K tile last releases it
        auto issue_s = [&](int x, uint32_t pos, bool first_, bool release_k, bool last) {
            bool good = true;
            if (first_) good = WAIT_ALL(&q_full[x], qn[x]++ & 1, 0x510);
            good = good && kv_wait(pos, 0x511);
            if (!good) return false;
            tc_fence_after();
            const uint64_t q = dQ0 + (uint32_t)x * TILE_UNITS, k = dK0 + (pos % RING) * TILE_UNITS;
            if (leader) {
                #pragma unroll
                for (int kk = 0; kk < 8; kk++)
                    if (kk < ks)
                        umma_ss(tmem_base + x * 128, q + (kk >> 2) * CHUNK_UNITS + (kk & 3) * 2, k + (kk >> 2) * CHUNK_UNITS + (kk & 3) * 2, idesc_s, kk > 0);
                umma_commit(&s_full[x]);
                if (release_k) umma_commit(&kv_empty[pos % RING]);
                if (last) umma_commit(&q_empty[x]);
            }
            return true;
        };
        // O_x += P_x V: A = P_x in TMEM (16 keys = 8 columns per step), B = V N-major (16 rows = 2048 bytes per step)
        auto issue_pv = [&](int x, uint32_t pos, bool first_, bool release_v, bool last) {
            bool good = kv_wait(pos, 0x515) && WAIT_ALL(&p_ready[x], tp[x] & 1, 0x514);
            if (good && first_ && on[x] > 0) good = WAIT_ALL(&o_free[x], (on[x] - 1) & 1, 0x517);
            if (!good) return false;
            tc_fence_after();
            const uint64_t v = dV0 + (pos % RING) * TILE_UNITS;
            if (leader) {
                #pragma unroll
                for (int kk = 0; kk < P_FIRST / 16; kk++) umma_ts(tmem_base + 256 + x * 128, tmem_base + x * 128 + kk * 8, v + 128 * kk, idesc_o, !first_ || kk > 0);
            }
            if (!WAIT_ALL(&p_rest[x], tp[x] & 1, 0x519)) return false;
            tc_fence_after();
            if (leader) {
                #pragma unroll
                for (int kk = P_FIRST / 16; kk < BT / 16; kk++) umma_ts(tmem_base + 256 + x * 128, tmem_base + x * 128 + kk * 8, v + 128 * kk, idesc_o, true);
                if (release_v) umma_commit(&kv_empty[pos % RING]);
                if (last) umma_commit(&o_full[x]);
            }
            tp[x]++;
            if (first_) on[x]++;
            return true;
        };
        // S_x(0) of a piece whose key tiles start at kabs_
        auto issue_first = [&](const WideItem& it, int x, uint32_t kabs_) { return issue_s(x, 2 * kabs_, true, x == it.has_b, it.n == 1); };
        WideItem im, nx;
        bool ok = take(0, im);
        if (ok) ok = issue_first(im, 0, 0);
        if (ok && im.has_b) ok = issue_first(im, 1, 0);
        for (uint32_t i = 0; ok && im.n > 0; i++) {
            const bool more = take(i + 1, nx);
            for (int j = 0; j < im.n && ok; j++) {
                const uint32_t kpos = 2 * (kabs + j);
                const bool last = j == im.n - 1;
                if (last && im.clean) {
                    ok = kv_wait(kpos + 1, 0x516);
                    if (ok && leader) mbar_arrive(v_here);
                    ok = ok && WAIT_ALL(v_clean, cleaned++ & 1, 0x518);
                }
                if (ok) ok = issue_pv(0, kpos + 1, j == 0, !im.has_b, last);
                if (ok && !last) ok = issue_s(0, kpos + 2, false, !im.has_b, j + 1 == im.n - 1);
                // the next piece's first S of slot A: its K tile is behind this piece's tiles in the ring
                if (ok && last && more) ok = issue_first(nx, 0, kabs + im.n);
                if (ok && im.has_b) {
                    ok = issue_pv(1, kpos + 1, j == 0, true, last);
                    if (ok && !last) ok = issue_s(1, kpos + 2, false, true, j + 1 == im.n - 1);
                }
            }
            kabs += im.n;
            if (ok && more && nx.has_b) ok = issue_first(nx, 1, kabs);
            give_back(i);
            im = nx;
        }
#undef WAIT_ALL
    }
    } else {
        regs_grow<REGS_HIGH>();
        // ---------------------------------------------------------------- softmax of slot x: thread = query row r of the slot's tile
        const int x = (warp - 4) >> 2;
        const int q4 = warp & 3;
        const int r = q4 * 32 + lane;
        const uint32_t lane_off = (uint32_t)(q4 * 32) << 16;
        const uint32_t tS = tmem_base + x * 128 + lane_off, tO = tmem_base + 256 + x * 128 + lane_off;
        const float cs = a.scale_log2e;
        const int tr = r / a.G, head = r - tr * a.G;       // token of the tile, query head of the cached one
        const float lag = 8.0f / cs;                       // how far a maximum may be ahead of the one that the probabilities refer to
        uint32_t t = 0, pieces = 0;                        // tiles, pieces of this slot so far
        bool ok = true;
        for (uint32_t i = 0; ok; i++) {
            if (!__all_sync(0xffffffffu, mbar_wait_relaxed(&item_full[i % QUEUE], (i / QUEUE) & 1, abort_flag, status, 0x533))) break;
            const volatile WideItem& it = queue[i % QUEUE];
            const int nj = it.n, j0 = it.j0, keys = it.keys, count = it.count;
            if (nj == 0) break;
            if (x == 1 && !it.has_b) { give_back(i); continue; }
            const int token = it.token + x * a.tokens + tr;
            const bool live = tr < a.tokens && token < count;
            const int context = keys - count;
            unsigned long long bits = 0;
            int limit = 0;                                 // keys [0, limit) are visible; with a tree, others behind them
            if (live && !(a.p.tree && count > 64)) {
                limit = a.p.tree ? context : min(keys, max(0, context + token + 1));
                if (a.p.tree) bits = (unsigned long long)a.p.tree[it.first + token] & (count < 64 ? (1ull << count) - 1 : ~0ull);
            }
            float m = -INFINITY, l = 0.f;                  // reference maximum (raw score units) and row sum relative to it
            for (int j = 0; j < nj; j++, t++) {
                ok = mbar_wait(&s_full[x], t & 1, abort_flag, status, 0x520 + x) && ok;
                tc_fence_after();
                uint32_t sv[128];
                tmem_ld32(tS, sv);
                tmem_ld32(tS + 32, sv + 32);
                tmem_ld32(tS + 64, sv + 64);
                tmem_ld32(tS + 96, sv + 96);
                tmem_ld_wait();
                const int rel = limit - (j0 + j) * BT;     // visible keys of this tile
                if (__any_sync(0xffffffffu, rel < BT)) {
                    uint32_t w[4];
                    #pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int lowest = rel - 32 * k;
                        w[k] = lowest >= 32 ? 0xffffffffu : lowest <= 0 ? 0u : (1u << lowest) - 1;
                        // bit i of the row's mask stands for key context + i: `lowest` + i of these 32
                        if (bits) w[k] |= lowest >= 32 || lowest <= -64 ? 0u : lowest >= 0 ? (uint32_t)(bits << lowest) : (uint32_t)(bits >> -lowest);
                    }
                    #pragma unroll
                    for (int e = 0; e < 128; e++) if (!(w[e >> 5] >> (e & 31) & 1u)) sv[e] = 0xff800000u;      // -inf
                }
                float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
                #pragma unroll
                for (int e = 0; e < 128; e += 8) {
                    mx0 = max3(mx0, __uint_as_float(sv[e]), __uint_as_float(sv[e + 1]));
                    mx1 = max3(mx1, __uint_as_float(sv[e + 2]), __uint_as_float(sv[e + 3]));
                    mx2 = max3(mx2, __uint_as_float(sv[e + 4]), __uint_as_float(sv[e + 5]));
                    mx3 = max3(mx3, __uint_as_float(sv[e + 6]), __uint_as_float(sv[e + 7]));
                }
                const float mx = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3));
                // a moved maximum rescales the row sum now and the row of O_X below (decided per warp, so that the TMEM accesses stay
                // warp-wide)
                const bool moved = __any_sync(0xffffffffu, mx > m + lag || (m == -INFINITY && mx > m)) != 0;
                float alpha = 1.0f;
                if (moved) {
                    const float m_new = fmaxf(m, mx);
                    alpha = m == -INFINITY ? 0.f : ex2_fast((m - m_new) * cs);
                    l *= alpha;
                    m = m_new;
                }
                const float moff = m == -INFINITY ? 0.f : m * cs;      // no key seen yet: every probability below is 2^-inf = 0
                const uint64_t cs2 = f2_both(cs), moff2 = f2_both(-moff);
                if (moved && j > 0) {                       // O_X(t-1) is complete: its product was issued ahead of S_X(t)
                    #pragma unroll
                    for (int cc = 0; cc < 4; cc++) {
                        if (cc * 2 < a.ks) {
                            uint32_t ov[32];
                            tmem_ld32(tO + cc * 32, ov);
                            tmem_ld_wait();
                            #pragma unroll
                            for (int e = 0; e < 32; e++) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
                            tmem_st32(tO + cc * 32, ov);
                        }
                    }
                }
                uint64_t rs0 = 0, rs1 = 0;
                // P goes back in two parts, over this row's own scores: the product begins with the first
                #pragma unroll
                for (int part = 0; part < 2; part++) {
                    const int e0 = part ? P_FIRST : 0, e1 = part ? BT : P_FIRST;
                    uint32_t pk[64];
                    #pragma unroll
                    for (int e = e0; e < e1; e += 4) {
                        const float2 x0 = f2_unpack(f2_fma(f2_pack_u(sv[e], sv[e + 1]), cs2, moff2)), x1 = f2_unpack(f2_fma(f2_pack_u(sv[e + 2], sv[e + 3]), cs2, moff2));
                        const float2 q0 = make_float2(ex2_fast(x0.x), ex2_fast(x0.y));
                        const float2 q1 = make_float2(ex2_fast(x1.x), ex2_fast(x1.y));
                        rs0 = f2_add(rs0, f2_pack(q0.x, q0.y));
                        rs1 = f2_add(rs1, f2_pack(q1.x, q1.y));
                        pk[e >> 1] = pack_bf16x2(q0.x, q0.y);
                        pk[(e >> 1) + 1] = pack_bf16x2(q1.x, q1.y);
                    }
                    #pragma unroll
                    for (int w = e0 >> 1; w < e1 >> 1; w += 16) tmem_st16(tS + w, pk + w);
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(part ? &p_rest[x] : &p_ready[x]);
                }
                const float2 rs = f2_unpack(f2_add(rs0, rs1));
                l += rs.x + rs.y;
            }
            // ---- end of the piece
            ok = mbar_wait(&o_full[x], pieces & 1, abort_flag, status, 0x528 + x) && ok;
            pieces++;
            tc_fence_after();
            const bool whole = it.whole;
            m = paged_maximum(m, limit, bits, count, keys);
            const float inv = paged_inverse(m, l);
            bf16* orow = a.p.out + (size_t)(it.first + (live ? token : 0)) * a.p.ldo + (it.g * a.G + head) * c.hs;
            float* part = wide_part(a.p.ws, gridDim.x, c.hs, it.part, 4 * x + q4) + lane;
            #pragma unroll
            for (int cc = 0; cc < 4; cc++) {
                if (cc * 2 < a.ks) {
                    uint32_t ov[32];
                    tmem_ld32(tO + cc * 32, ov);
                    tmem_ld_wait();
                    if (live && ok) {
                        #pragma unroll
                        for (int u = 0; u < 4; u++) {
                            const int ch = cc * 32 + u * 8;
                            if (ch < c.hs) {
                                if (whole) {
                                    uint4 o;
                                    o.x = pack_bf16x2(__uint_as_float(ov[8 * u]) * inv, __uint_as_float(ov[8 * u + 1]) * inv);
                                    o.y = pack_bf16x2(__uint_as_float(ov[8 * u + 2]) * inv, __uint_as_float(ov[8 * u + 3]) * inv);
                                    o.z = pack_bf16x2(__uint_as_float(ov[8 * u + 4]) * inv, __uint_as_float(ov[8 * u + 5]) * inv);
                                    o.w = pack_bf16x2(__uint_as_float(ov[8 * u + 6]) * inv, __uint_as_float(ov[8 * u + 7]) * inv);
                                    *reinterpret_cast<uint4*>(orow + ch) = o;
                                } else {
                                    #pragma unroll
                                    for (int e = 0; e < 8; e++) part[(ch + e) * 32] = __uint_as_float(ov[8 * u + e]);
                                }
                            }
                        }
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_free[x]);            // O_X may be overwritten by the next piece's first product
            if (live && ok && !whole) { part[c.hs * 32] = m == -INFINITY ? m : m * cs; part[(c.hs + 1) * 32] = l; }
            give_back(i);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (*abort_flag) {
        long long t0 = clock64();
        while (clock64() - t0 < 2000000ll) { __nanosleep(1000); }
        __syncthreads();
    }
    if (warp == 1) tmem_dealloc(tmem_base, TMEM_COLS);
}

constexpr int JOIN_CHANNELS = 16;

// Joins the parts of a piece that lies in several shares: a block for 32 rows of it, a warp for 16 channels, a lane for a row; two partials are on their way at a time
__global__ void __launch_bounds__(256)
paged_wide_join_kernel(const PagedAttention a, int blocks, int hs, int G, int tokens) {
    const int k = blockIdx.x + 1, group = blockIdx.y, lane = threadIdx.x & 31, ch0 = (threadIdx.x >> 5) * JOIN_CHANNELS;
    pdl_wait();                                                // the parts
    pdl_trigger();
    const PagedJoin* joins = reinterpret_cast<const PagedJoin*>(a.ws);
    const int parts = joins[k].parts;
    if (parts == 0 || ch0 >= hs) return;
    const int r = (group & 3) * 32 + lane, tr = r / G, token = joins[k].row + (group >> 2) * tokens + tr, first = joins[k].first, g = joins[k].g;
    if (tr >= tokens || token >= joins[k].count) return;
    float m = -INFINITY, l = 0.f, acc[JOIN_CHANNELS] = {};
    for (int j0 = 0; j0 < parts; j0 += 2) {
        float mj[2], lj[2], v[2][JOIN_CHANNELS];
        #pragma unroll
        for (int q = 0; q < 2; q++) {
            const int j = min(j0 + q, parts - 1);              // past the last one: again, with no weight
            const float* p = wide_part(a.ws, blocks, hs, 2 * (k - 1 + j) + (j == 0), group) + lane;
            mj[q] = j0 + q < parts ? p[hs * 32] : -INFINITY;
            lj[q] = p[(hs + 1) * 32];
            #pragma unroll
            for (int e = 0; e < JOIN_CHANNELS; e++) v[q][e] = ch0 + e < hs ? p[(ch0 + e) * 32] : 0.f;
        }
        const float mn = fmaxf(m, fmaxf(mj[0], mj[1])), ref = mn == -INFINITY ? 0.f : mn;
        const float ca = ex2_fast(m - ref), c0 = ex2_fast(mj[0] - ref), c1 = ex2_fast(mj[1] - ref);
        l = fmaf(lj[0], c0, fmaf(lj[1], c1, l * ca));
        #pragma unroll
        for (int e = 0; e < JOIN_CHANNELS; e++) acc[e] = fmaf(v[0][e], c0, fmaf(v[1][e], c1, acc[e] * ca));
        m = mn;
    }
    const float inv = paged_inverse(m, l);
    bf16* out = a.out + (size_t)(first + token) * a.ldo + (g * G + (r - tr * G)) * hs + ch0;
    #pragma unroll
    for (int u = 0; u < JOIN_CHANNELS / 8; u++)
        if (ch0 + u * 8 < hs)
            *reinterpret_cast<uint4*>(out + u * 8) = make_uint4(pack_bf16x2(acc[8 * u] * inv, acc[8 * u + 1] * inv), pack_bf16x2(acc[8 * u + 2] * inv, acc[8 * u + 3] * inv),
                                                                pack_bf16x2(acc[8 * u + 4] * inv, acc[8 * u + 5] * inv), pack_bf16x2(acc[8 * u + 6] * inv, acc[8 * u + 7] * inv));
}

// A bound of the number of units, from what the host knows
long long wide_units(const PagedCache* c, int N, int NH) {
    const int G = NH / c->heads, step = 2 * (BT / G);
    const long long keys = (long long)c->table_width << c->page_shift;
    return (CEIL_DIV((long long)N, step) + c->sequences) * c->heads * (CEIL_DIV(keys, BT) + 4);
}
int wide_blocks(const PagedCache* c, int N, int NH) {
    int sms = llmc_device_sm_count(); if (sms <= 0) sms = 148;
    const long long units = wide_units(c, N, NH);
    return (int)(units < sms ? units : sms);
}

}  // namespace

// The rows of a sequence on average decide for the whole call, so that where single tokens stand beside one part of a prompt one of the two is in the wrong place (us, single tokens alone, the part
// alone, both in one call: 31 of up to 8192 keys and a part of 2048 tokens 97, 59, 170; 127 of up to 4000 and a part of 384 behind 8000 keys 183, 62, 601).
// Whether row tiles take a call, or groups of 16 rows, which read a sequence's keys once for each group, but begin and end sooner and have more pieces to go round: by the rows of a sequence and
// cached head, on average.  us, row tiles / groups: heads of 128, 14 rows of 32 sequences of up to 4000 keys 81 / 81, 18 rows 81 / 83, 27 rows 82 / 109, 24 rows of 8 of 2000 27.4 / 28.4; heads of 64,
// 26 rows of 32 of up to 1024 43 / 41.5, 35 rows 43 / 50, 24 rows of 8 of 2000 23.6 / 21.8, 36 rows 23.9 / 26.4.  Where the groups have an SM each and the table has room
// for few keys they are ahead for longer: 48 rows of one sequence of 1500 16.2 / 13.9, 32 rows of one of 8000 26.8 / 21, 48 rows 27.7 / 27.6, 64 rows 27 / 33, 43 rows of 4 of 300 14.9 / 13.2; heads of
// 64, 48 rows of one of 8000 23.5 / 21.6, 64 rows 23.2 / 24.5.  With more keys, 32 rows: one of 32000 45 / 51, of 100000 97 / 137, 28 rows of 4 of 16000 65 / 80, 32 cached heads of 8000 41 / 53.
bool paged_wide(const PagedCache* c, int N, int NH) {
    int sms = llmc_device_sm_count(); if (sms <= 0) sms = 148;
    const int G = NH / c->heads;
    const long long room = ((long long)c->table_width << c->page_shift) * c->sequences * c->heads;
    const long long most = paged_few_pieces(c, N, NH, 16) <= sms && room <= 1000LL * sms ? 48 : c->hs > 64 ? 16 : 24;
    return G <= BT && ((long long)N * G > most * c->sequences || !paged_few_fits(c, N, NH));
}

long long paged_wide_workspace(const PagedCache* c, int N, int NH) { return wide_blocks(c, N, NH) * ((long long)sizeof(PagedJoin) / 4 + 4LL * BT * (c->hs + 2)); }

// (a piece of one tile is not cut)
int paged_wide_launches(const PagedCache* c, int N, int NH) { return wide_blocks(c, N, NH) > 1 && ((long long)c->table_width << c->page_shift) > BT ? 2 : 1; }

int paged_wide_launch(const PagedCache* c, const PagedAttention& p, cudaStream_t stream) {
    WideArgs a;
    a.p = p;
    a.G = p.NH / c->heads;
    a.tokens = BT / a.G;
    a.ks = CEIL_DIV(c->hs, 16);
    const int step = 2 * a.tokens;
    a.by_step = FastDiv(step);
    for (a.period_log2 = 0; step % (BT >> a.period_log2); ) a.period_log2++;
    a.rise = (step << a.period_log2) / BT;
    a.new_tiles[0] = 0;
    for (int i = 1; i <= 1 << a.period_log2; i++) a.new_tiles[i] = (unsigned short)(a.new_tiles[i - 1] + CEIL_DIV(i * step, BT));
    // (us, counted as nothing / one / two / three units: prompt of 8192 tokens 657 / 605 / 587 / 583, 16 trees of up to 64 tokens 84 / 69 / 68 / 69, prompt of 777 28 / 26 / 25 / 26)
    a.over = 2;
    a.box = (1 << c->page_shift) < BT ? 1 << c->page_shift : BT;
    a.scale_log2e = 1.0f / sqrtf((float)c->hs) * 1.4426950408889634f;
    CUtensorMap tmQ, tmK, tmV;
    const uint64_t hs = c->hs;
    {
        uint64_t dims[3] = {hs, (uint64_t)p.NH, (uint64_t)p.N}, strides[3] = {2, hs * 2, (uint64_t)p.ldq * 2};
        uint32_t box[3] = {64, (uint32_t)a.G, (uint32_t)a.tokens};
        const int bad = llmc_get_tensormap(&tmQ, p.q, 2, 3, dims, strides, box, 3);
        if (bad) return bad;
    }
    int rc = paged_maps(&tmK, &tmV, c, p.layer, a.box);
    if (rc) return rc;
    static bool done[64];
    rc = paged_shared_memory(paged_wide_kernel, SMEM, done);
    if (rc) return rc;
    if (wide_units(c, p.N, p.NH) >= PAGED_UNITS) return -7;
    const int blocks = wide_blocks(c, p.N, p.NH);
    CUDA_CHECK(launch_pdl(paged_wide_kernel, dim3(blocks), dim3(THREADS), SMEM, stream, 0, tmQ, tmK, tmV, *c, a));
    if (paged_wide_launches(c, p.N, p.NH) > 1) CUDA_CHECK(launch_pdl(paged_wide_join_kernel, dim3(blocks - 1, 8), dim3(256), 0, stream, 0, a.p, blocks, c->hs, a.G, a.tokens));
    return 0;
}
