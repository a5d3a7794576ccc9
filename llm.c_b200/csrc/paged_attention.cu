// Attention of ragged new tokens over a key / value cache in pages (paged.cuh):
//
//   out[n, h] = sum over the keys s that row n sees of softmax_s(q[n, h] . K[s, g] / sqrt(HS)) V[s, g],  g = h / (NH / NKV); 0 where it sees none.
//   Token i of a sequence of `len` keys with `count` new ones sees slots 0 .. len - count + i; with `tree` it sees slots below len - count, and slot len - count + j
//   where bit j of tree[n] is set (at most 64 new tokens of a sequence).
//
// Few rows to a cached head (a decoding step): reading the cache once is all the work there is.  A piece is one cached head of one sequence for 8 query rows (its tokens' grouped heads), or 16.
//   * Every warp has a share of the keys of its own (COOP = 1): no warp waits for another.  Where there are not many pieces a block's four warps share the keys of a piece and merge
//     their sums in shared memory (COOP = 4).  Parts of a piece that lie in several shares are joined by a second kernel; where no sequence can have more than 256 keys there are none.
//   * Tiles of 16 keys arrive by TMA through a ring of the warp's own, 2 to 4 copies a tile (a page, or 16 rows of a larger one, by 64 channels).  The next 32 tiles' pages are looked up at
//     once, a lane for each, so that no copy waits for the table.  (With cp.async, a lane for each 16 bytes, the addresses took most of the instructions.)
//   * The copies run ahead of the arithmetic across the ends of pieces.
//   * S = Q K^T and O += P V on warp-level MMAs, the query rows as the 16-row operand.  P keeps 16 bits: the upper 8 as a bf16, the next 8 as another; with 8 rows the second one takes the
//     operand's idle rows 8..15, and the two halves of the accumulator are added at the end.  (One bf16 would leave an error as large as the output's rounding.)
//   * Slots behind the length may hold anything: scores there are replaced, and the values in the last tile are overwritten with zeros in shared memory before the product reads them.
#include "paged_attention_ops.h"
#include "pdl.cuh"

namespace {

constexpr int PF_WARPS = 4;
constexpr int PF_THREADS = PF_WARPS * 32;
constexpr int PF_TILE = 16;           // keys per tile of a warp
constexpr float PF_LOG2E = 1.4426950408889634f;

DEVINL void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
DEVINL void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
DEVINL void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
DEVINL uint32_t top_bf16x2(float lo, float hi) { return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632); }     // bf16 without rounding

struct FewArgs : PagedAttention {
    int unit_log2;             // keys of a unit: 16 at least
    int over;                  // units that a piece counts besides its keys: what it takes to begin and to end one
    int box;                   // rows of a page that one copy brings, 8 or 16
    float scale_log2e;
};

template <int HS_> __host__ __device__ constexpr int pf_stages() { return HS_ == 64 ? 6 : 3; }              // 96 KB a block: two blocks on an SM
template <int HS_> __host__ __device__ constexpr int pf_stage_bytes() { return 2 * PF_TILE * HS_ * 2; }    // K tile, V tile
template <int HS_, int ROWS> __host__ __device__ constexpr int pf_part_floats() { return ROWS * (HS_ + 2); }
template <int HS_, int COOP> __host__ __device__ constexpr int pf_smem_bytes() {
    return PF_WARPS * (pf_stages<HS_>() * (pf_stage_bytes<HS_>() + 8) + (COOP > 1 ? pf_part_floats<HS_, 8>() * 4 : 0)) + 8;         // rings and their barriers, partials of 8 rows, flag
}

// The pieces of a sequence, head by head, and in a head by groups of ROWS query rows: row r is token r / G, head g G + r % G
template <int ROWS>
struct FewUnits {
    const PagedCache& c;
    const FewArgs& a;
    int G;
    DEVINL PagedSpan span(int b) const { return paged_span(c, b, a.N, a.status, 0x48); }
    DEVINL int groups(const PagedSpan& s) const { return (s.count * G + ROWS - 1) / ROWS; }
    DEVINL int tiles(const PagedSpan& s) const { return s.keys > 0 ? ((s.keys - 1) >> a.unit_log2) + 1 : 1; }
    DEVINL int operator()(const PagedSpan& s) const { return groups(s) * c.heads * (a.over + tiles(s)); }
};

// The pieces of a share that it has keys of, one after the other
template <int ROWS>
struct FewWalk {
    PagedSpan s;
    int b, g, grp, ng, nt;     // groups, units of keys of a piece
    int t0, t1;                // units of this piece's keys that lie in the share
    int left;                  // units of the share behind this piece
    // begins `units` units at p; false: they hold no keys
    DEVINL bool start(const FewUnits<ROWS>& u, const PagedPlace& p, int units) {
        b = p.b; s = p.s; ng = u.groups(s); nt = u.tiles(s);
        if (ng == 0) return false;
        const int piece = p.offset / (nt + u.a.over), x = p.offset - piece * (nt + u.a.over) - u.a.over;
        g = piece / ng;
        grp = piece - g * ng;
        t0 = max(0, x);
        t1 = min(nt, x + units);
        left = units - (min(nt, x + units) - x);
        return t1 > t0 || next(u);
    }
    DEVINL bool next(const FewUnits<ROWS>& u) {
        if (left <= u.a.over) return false;
        if (++grp == ng) {
            grp = 0;
            if (++g == u.c.heads) {
                g = 0;
                do {
                    if (++b >= u.c.sequences) return false;
                    s = u.span(b);
                    ng = u.groups(s);
                } while (ng == 0);
                nt = u.tiles(s);
            }
        }
        t0 = 0;
        t1 = min(nt, left - u.a.over);
        left -= u.a.over + t1;
        return true;
    }
    // keys of this part; none of a sequence with more new tokens than a mask has bits
    DEVINL bool refused(const FewArgs& a) const { return a.tree && s.count > 64; }
    DEVINL int k0(const FewArgs& a) const { return t0 << a.unit_log2; }
    DEVINL int k1(const FewArgs& a) const { return refused(a) ? 0 : min(s.keys, t1 << a.unit_log2); }
};

// The workspace: what is to be joined, for each share; two partials for each share, ROWS x (HS_ + 2) words each
DEVINL float* few_parts(float* ws, int shares) { return ws + shares * (sizeof(PagedJoin) / 4); }

template <int HS_, int ROWS, int COOP>
__global__ void __launch_bounds__(PF_THREADS, 2)
paged_few_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const PagedCache c, const FewArgs a) {
    constexpr int CH = HS_ / 64;               // 64-channel chunks: 16 rows of 128 bytes, 128-byte swizzled
    constexpr int KS = HS_ / 16;               // 16-channel steps
    constexpr int STAGES = pf_stages<HS_>();
    constexpr int STAGE = pf_stage_bytes<HS_>(), VALUES = STAGE / 2;
    constexpr int PART = pf_part_floats<HS_, ROWS>(), MERGE = pf_part_floats<HS_, 8>();
    constexpr int H = ROWS / 8;                // rows gq + 8 h of this lane
    constexpr int TEAMS = PF_WARPS / COOP;     // shares of a block
    constexpr int STEP = COOP * PF_TILE;
    extern __shared__ __align__(1024) uint8_t pf_smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int gq = lane >> 2, tq4 = lane & 3;                  // MMA fragment coordinates: row gq, column pair tq4
    uint8_t* ring = pf_smem + warp * (STAGES * STAGE);
    float* merge = reinterpret_cast<float*>(pf_smem + PF_WARPS * STAGES * STAGE);
    uint64_t* full_bars = reinterpret_cast<uint64_t*>(merge + (COOP > 1 ? PF_WARPS * MERGE : 0));
    uint64_t* full = full_bars + warp * STAGES;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(full_bars + PF_WARPS * STAGES);
    if (threadIdx.x == 0) {
        for (int i = 0; i < PF_WARPS * STAGES; i++) mbar_init(&full_bars[i], 1);
        *abort_flag = 0;
        mbar_fence_init();
        tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV);
    }
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    const int hs = c.hs, G = a.NH / c.heads;
    const FewUnits<ROWS> units{c, a, G};
    const int most = gridDim.x * TEAMS, share = blockIdx.x * TEAMS + warp / COOP, member = warp % COOP;
    PagedPlace place;
    const PagedShares shares(paged_find(c, a.N, a.status, 0x48, units, [&](int sum) {
        const PagedShares sh(sum, most);
        return share < sh.blocks ? sh.first(share) : -1;
    }, place), most);
    PagedJoin* join = reinterpret_cast<PagedJoin*>(a.ws) + share;
    const bool notes = member == 0 && lane == 0;
    if (share >= shares.blocks) { if (notes) join->parts = 0; return; }
    const int first = shares.first(share), count = shares.first(share + 1) - first;
    FewWalk<ROWS> w, f;                                        // what is worked on, what is fetched
    if (!w.start(units, place, count)) { if (notes) join->parts = 0; return; }
    f = w;
    // query rows; the A operand of S: lane holds channels 2 tq4, 2 tq4 + 1 and + 8, + 9 of row gq.  Rows past the piece's are zero and dropped at the end.
    uint32_t qa[KS][2 * H];
    unsigned long long bits[H];
    int limit[H];                                              // keys [0, limit) are visible to the row; with a tree, others behind them
    auto load_rows = [&]() {
        const int rows = min(ROWS, w.s.count * G - w.grp * ROWS), context = w.s.keys - w.s.count, k1 = w.k1(a);
        #pragma unroll
        for (int h = 0; h < H; h++) {
            const bool in = gq + 8 * h < rows;
            const int r = w.grp * ROWS + (in ? gq + 8 * h : 0), token = r / G;
            const bf16* qr = a.q + (w.s.first + token) * a.ldq + (w.g * G + r - token * G) * hs + 2 * tq4;
            #pragma unroll
            for (int kk = 0; kk < KS; kk++) {
                qa[kk][h] = in && kk * 16 < hs ? *reinterpret_cast<const uint32_t*>(qr + kk * 16) : 0u;
                qa[kk][H + h] = in && kk * 16 + 8 < hs ? *reinterpret_cast<const uint32_t*>(qr + kk * 16 + 8) : 0u;
            }
            bits[h] = a.tree ? (unsigned long long)a.tree[w.s.first + token] : 0;
            limit[h] = min(k1, a.tree ? context : context + token + 1);
        }
    };
    load_rows();

    // ---- the warp's copies
    int fkt = f.k0(a) + member * PF_TILE, fk1 = f.k1(a);
    int look = fkt - 32 * STEP, page_lo = 0, page_hi = 0;   // pages of 32 tiles from key `look` on, a lane for each; of 8-row pages a tile has two
    bool more = true;
    auto fetch = [&](int st) {
        while (more && fkt >= fk1) {
            more = f.next(units);
            fkt = f.k0(a) + member * PF_TILE;
            fk1 = f.k1(a);
            look = fkt - 32 * STEP;
        }
        if (!more) return;
        if (fkt >= look + 32 * STEP) {
            look = fkt;
            const int slot = fkt + lane * STEP;
            // a page that is not there lies outside the tensor map: zeros
            auto page_of = [&](int sl) { int p = -1; if (sl < fk1) p = paged_page(c, f.b, sl, a.status, 0x4A); return p < 0 ? c.pages : p; };
            page_lo = page_of(slot);
            page_hi = a.box == 8 ? page_of(slot + 8) : 0;
        }
        const int from = (fkt - look) / STEP;
        const int p0 = __shfl_sync(0xffffffffu, page_lo, from), p1 = __shfl_sync(0xffffffffu, page_hi, from);
        if (lane == 0) {
            uint8_t* dst = ring + st * STAGE;
            const int row = fkt & ((1 << c.page_shift) - 1);
            mbar_expect_tx(&full[st], STAGE);
            #pragma unroll
            for (int ch = 0; ch < CH; ch++) {
                tma_load_4d(dst + ch * 2048, &tmK, &full[st], ch * 64, f.g, row, p0);
                tma_load_4d(dst + VALUES + ch * 2048, &tmV, &full[st], ch * 64, f.g, row, p0);
                if (a.box == 8) {
                    tma_load_4d(dst + ch * 2048 + 1024, &tmK, &full[st], ch * 64, f.g, 0, p1);
                    tma_load_4d(dst + VALUES + ch * 2048 + 1024, &tmV, &full[st], ch * 64, f.g, 0, p1);
                }
            }
        }
        fkt += STEP;
    };
    for (int st = 0; st < STAGES; st++) fetch(st);
    if (notes) {
        const int tile0 = first + count - w.left - w.t1;       // where unit 0 of the piece's keys lies among all units
        const bool mine = w.t0 > 0 && shares.share_of(tile0) == share - 1;     // inside the piece, and the first share that begins there
        *join = {mine ? shares.share_of(tile0 + w.nt - 1) - share + 2 : 0, w.s.first, w.s.count, w.g, w.grp * ROWS};
    }

    const float sl2 = a.scale_log2e;
    const int mrow = lane & 7, mid = lane >> 3;                // ldmatrix: lane supplies the row address of matrix lane / 8, row lane % 8
    int st = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (bool again = true; again;) {
        const int rows = min(ROWS, w.s.count * G - w.grp * ROWS);
        const int context = w.s.keys - w.s.count, k1 = w.k1(a);
        if (w.refused(a) && notes) record_error(a.status, ST_BAD_ARG, 0x49);
        float m[H], l[H];                                      // of row gq + 8 h; l: this lane's keys only
        #pragma unroll
        for (int h = 0; h < H; h++) { m[h] = -INFINITY; l[h] = 0.f; }
        float acc[HS_ / 8][4];                                 // columns 2 tq4, + 1 of channel group n: [0,1] of row gq; [2,3] of row gq + 8, or of row gq from the lower bits of P
        #pragma unroll
        for (int n = 0; n < HS_ / 8; n++) { acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f; }
        for (int kt = w.k0(a) + member * PF_TILE; kt < k1; kt += STEP) {
            ok = __all_sync(0xffffffffu, mbar_wait(&full[st], phase, abort_flag, a.status, 0x540)) && ok;
            const uint32_t kb = smem_u32(ring + st * STAGE), vb = kb + VALUES;
            if (kt + PF_TILE > w.s.keys) {                     // the sequence's last tile
                for (int i = (w.s.keys - kt) * 8 + lane; i < PF_TILE * 8; i += 32)
                    #pragma unroll
                    for (int ch = 0; ch < CH; ch++) *reinterpret_cast<uint4*>(ring + st * STAGE + VALUES + ch * 2048 + i * 16) = make_uint4(0, 0, 0, 0);
                fence_async_smem();                            // (the stage's next copy comes behind these stores)
                __syncwarp();
            }
            // ---- S (rows gq, gq + 8; keys 2 tq4 + {0,1} of each group of 8 keys)
            float sc[2][4];
            #pragma unroll
            for (int k = 0; k < 2; k++) { sc[k][0] = sc[k][1] = sc[k][2] = sc[k][3] = 0.f; }
            #pragma unroll
            for (int kk = 0; kk < KS; kk++) {
                uint32_t kf[4];     // matrices: keys 0-7 channels 0-7 / 8-15 of the step, keys 8-15 likewise
                const int row = (mid >> 1) * 8 + mrow, ch = kk * 2 + (mid & 1);
                ldmatrix4(kf, kb + (ch >> 3) * 2048 + row * 128 + (((ch & 7) ^ (row & 7)) * 16));
                mma_16x8x16(sc[0], qa[kk][0], H == 2 ? qa[kk][1] : 0u, qa[kk][H], H == 2 ? qa[kk][H + 1] : 0u, kf[0], kf[1]);
                mma_16x8x16(sc[1], qa[kk][0], H == 2 ? qa[kk][1] : 0u, qa[kk][H], H == 2 ? qa[kk][H + 1] : 0u, kf[2], kf[3]);
            }
            // ---- running softmax (base 2); the four lanes of a row hold its 16 keys
            uint32_t hi[2][H], lo[2][H];
            float corr[H];
            #pragma unroll
            for (int h = 0; h < H; h++) {
                float sv[4];
                #pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int key = kt + (e >> 1) * 8 + 2 * tq4 + (e & 1);
                    bool seen = key < limit[h];
                    if (a.tree && key >= context) seen = key < k1 && (bits[h] >> (key - context) & 1);
                    sv[e] = seen ? sc[e >> 1][2 * h + (e & 1)] * sl2 : -INFINITY;
                }
                float mn = fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3]));
                mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 1));
                mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 2));
                mn = fmaxf(mn, m[h]);
                const float mref = mn == -INFINITY ? 0.f : mn; // no key seen yet: every probability below is 2^-inf = 0
                corr[h] = ex2_fast(m[h] - mref);
                float p[4];
                #pragma unroll
                for (int e = 0; e < 4; e++) p[e] = ex2_fast(sv[e] - mref);
                l[h] = l[h] * corr[h] + ((p[0] + p[1]) + (p[2] + p[3]));
                m[h] = mn;
                #pragma unroll
                for (int k = 0; k < 2; k++) {
                    hi[k][h] = top_bf16x2(p[2 * k], p[2 * k + 1]);
                    const float2 hf = unpack_bf16x2(hi[k][h]);
                    lo[k][h] = pack_bf16x2(p[2 * k] - hf.x, p[2 * k + 1] - hf.y);
                }
            }
            if (__any_sync(0xffffffffu, corr[0] != 1.0f || corr[H - 1] != 1.0f)) {
                #pragma unroll
                for (int n = 0; n < HS_ / 8; n++) { acc[n][0] *= corr[0]; acc[n][1] *= corr[0]; acc[n][2] *= corr[H - 1]; acc[n][3] *= corr[H - 1]; }
            }
            // ---- O += P V: 16 keys, 16 channels per ldmatrix
            #pragma unroll
            for (int n2 = 0; n2 < HS_ / 16; n2++) {
                uint32_t vf[4];     // matrices: keys 0-7 / 8-15 of channels 0-7 of the pair of groups, then of channels 8-15
                const int row = (mid & 1) * 8 + mrow, ch = n2 * 2 + (mid >> 1);
                ldmatrix4_trans(vf, vb + (ch >> 3) * 2048 + row * 128 + (((ch & 7) ^ (row & 7)) * 16));
                if (H == 1) {
                    mma_16x8x16(acc[2 * n2], hi[0][0], lo[0][0], hi[1][0], lo[1][0], vf[0], vf[1]);
                    mma_16x8x16(acc[2 * n2 + 1], hi[0][0], lo[0][0], hi[1][0], lo[1][0], vf[2], vf[3]);
                } else {
                    mma_16x8x16(acc[2 * n2], hi[0][0], hi[0][H - 1], hi[1][0], hi[1][H - 1], vf[0], vf[1]);
                    mma_16x8x16(acc[2 * n2 + 1], hi[0][0], hi[0][H - 1], hi[1][0], hi[1][H - 1], vf[2], vf[3]);
                    mma_16x8x16(acc[2 * n2], lo[0][0], lo[0][H - 1], lo[1][0], lo[1][H - 1], vf[0], vf[1]);
                    mma_16x8x16(acc[2 * n2 + 1], lo[0][0], lo[0][H - 1], lo[1][0], lo[1][H - 1], vf[2], vf[3]);
                }
            }
            __syncwarp();                                      // the stage may be refilled
            fetch(st);
            if (++st == STAGES) { st = 0; phase ^= 1; }
        }
        #pragma unroll
        for (int h = 0; h < H; h++) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            m[h] = paged_maximum(m[h], limit[h], k1 > 0 ? bits[h] : 0, w.s.count, w.s.keys);
        }
        // the next piece's rows are on their way while this one ends
        const FewWalk<ROWS> d = w;
        again = w.next(units);
        if (again) load_rows();
        const bool whole = d.t1 - d.t0 == d.nt;
        float* part = few_parts(a.ws, most) + (size_t)(2 * share + (d.t0 == 0)) * PART;
        auto out_row = [&](int r) { const int row = d.grp * ROWS + r, token = row / G; return a.out + (d.s.first + token) * a.ldo + (d.g * G + row - token * G) * hs; };
        if (COOP == 1) {
            #pragma unroll
            for (int h = 0; h < H; h++) {
                const int r = gq + 8 * h;
                if (r < rows) {
                    const float inv = paged_inverse(m[h], l[h]);
                    bf16* o = out_row(r) + 2 * tq4;
                    float* p = part + r * HS_ + 2 * tq4;
                    #pragma unroll
                    for (int n = 0; n < HS_ / 8; n++) {
                        const float x = H == 1 ? acc[n][0] + acc[n][2] : acc[n][2 * h], y = H == 1 ? acc[n][1] + acc[n][3] : acc[n][2 * h + 1];
                        if (!whole) *reinterpret_cast<float2*>(p + n * 8) = make_float2(x, y);
                        else if (n * 8 < hs) *reinterpret_cast<uint32_t*>(o + n * 8) = pack_bf16x2(x * inv, y * inv);
                    }
                    if (!whole && tq4 == 0) { part[ROWS * HS_ + r] = m[h]; part[ROWS * HS_ + ROWS + r] = l[h]; }
                }
            }
        } else {
            // merge the warps in warp order, 8 rows at a time; a row's groups of 8 channels change places, so that the rows of an accumulator fall into different banks
            float* wp = merge + warp * MERGE;
            #pragma unroll
            for (int h = 0; h < H; h++) {
                const int here = min(8, rows - 8 * h);
                if (here <= 0) break;
                #pragma unroll
                for (int n = 0; n < HS_ / 8; n++)
                    *reinterpret_cast<float2*>(wp + gq * HS_ + ((n * 8) ^ ((gq & 3) * 8)) + 2 * tq4) =
                        H == 1 ? make_float2(acc[n][0] + acc[n][2], acc[n][1] + acc[n][3]) : make_float2(acc[n][2 * h], acc[n][2 * h + 1]);
                if (tq4 == 0) { wp[8 * HS_ + gq] = m[h]; wp[8 * HS_ + 8 + gq] = l[h]; }
                __syncthreads();
                for (int i = threadIdx.x; i < here * (HS_ / 2); i += PF_THREADS) {
                    const int r = i / (HS_ / 2), ch = (i - r * (HS_ / 2)) * 2;
                    float mn = -INFINITY;
                    #pragma unroll
                    for (int v = 0; v < PF_WARPS; v++) mn = fmaxf(mn, merge[v * MERGE + 8 * HS_ + r]);
                    float x = 0.f, y = 0.f, ls = 0.f;
                    #pragma unroll
                    for (int v = 0; v < PF_WARPS; v++) {
                        const float mw = merge[v * MERGE + 8 * HS_ + r];
                        const float cw = (mw == -INFINITY) ? 0.f : ex2_fast(mw - mn);
                        const float2 o = *reinterpret_cast<const float2*>(merge + v * MERGE + r * HS_ + (ch ^ ((r & 3) * 8)));
                        x += o.x * cw;
                        y += o.y * cw;
                        ls += merge[v * MERGE + 8 * HS_ + 8 + r] * cw;
                    }
                    const float inv = paged_inverse(mn, ls);
                    if (!whole) {
                        *reinterpret_cast<float2*>(part + (8 * h + r) * HS_ + ch) = make_float2(x, y);
                        if (ch == 0) { part[ROWS * HS_ + 8 * h + r] = mn; part[ROWS * HS_ + ROWS + 8 * h + r] = ls; }
                    } else if (ch < hs) *reinterpret_cast<uint32_t*>(out_row(8 * h + r) + ch) = pack_bf16x2(x * inv, y * inv);
                }
                __syncthreads();                               // what comes next is merged in the same place
            }
        }
        again = again && !*abort_flag;
    }
    if (*abort_flag) {                                         // copies may still be on their way
        const long long t = clock64();
        while (clock64() - t < 2000000ll) __nanosleep(1000);
    }
}

// Joins the partials of pieces that lie in several shares.  A block looks at a share for each of its warps, and 32 channels.  A warp joins the piece that the first share inside it noted down, if it
// has few partials; of many, the block's warps take every PJ_WARPS-th each and are merged like the partials.  A lane has four channels of a row, or of a few, and four partials on their way at a
// time.  (Carried along by one thread from partial to partial, each load waits for the one before: one sequence of 2000 keys took 24 us instead of 20; with the shares worked out here again instead
// of read from the workspace, and the maxima read first, 11 instead of 9.)
// Blocks of four warps have room on an SM beside the kernel before, and start without a wait when it ends; eight are faster where pieces have many partials (us, four warps / eight: 32 sequences up
// to 8192 keys 107.3 / 109.2, 40 up to 4000 70.9 / 72.8; one of 2000 9.8 / 9.1, of 16000 20.8 / 20.0).
constexpr int PJ_CHANNELS = 32;
constexpr int PJ_ALONE = 8;            // partials that one warp joins by itself
template <int ROWS>
struct FewSum {
    static constexpr int R = ROWS / 4;         // rows of a lane: lane / 8 + 4 i
    float m[R], l[R];
    float4 acc[R];
    // partials j0, j0 + step, ... below `parts` of shares k - 1, k, ...
    template <int HS_>
    DEVINL void add(const float* base, int k, int parts, int rows, int j0, int step, int ch) {
        constexpr int PART = pf_part_floats<HS_, ROWS>();
        const int lane = threadIdx.x & 31;
        #pragma unroll
        for (int i = 0; i < R; i++) { m[i] = -INFINITY; l[i] = 0.f; acc[i] = make_float4(0.f, 0.f, 0.f, 0.f); }
        for (; j0 < parts; j0 += 4 * step) {
            float mj[4][R], lj[4][R];
            float4 v[4][R];
            #pragma unroll
            for (int q = 0; q < 4; q++) {
                const int j = j0 + q * step;
                const float* p = base + (size_t)(2 * (k - 1 + j) + (j == 0)) * PART;
                #pragma unroll
                for (int i = 0; i < R; i++) {
                    const int r = (lane >> 3) + 4 * i;
                    const bool in = j < parts && r < rows;
                    mj[q][i] = in ? p[ROWS * HS_ + r] : -INFINITY;
                    lj[q][i] = in ? p[ROWS * HS_ + ROWS + r] : 0.f;
                    v[q][i] = in ? *reinterpret_cast<const float4*>(p + r * HS_ + ch) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
            }
            #pragma unroll
            for (int i = 0; i < R; i++) {
                const float mn = fmaxf(fmaxf(fmaxf(mj[0][i], mj[1][i]), fmaxf(mj[2][i], mj[3][i])), m[i]), ref = mn == -INFINITY ? 0.f : mn;
                const float ca = ex2_fast(m[i] - ref);
                m[i] = mn;
                l[i] *= ca;
                acc[i].x *= ca; acc[i].y *= ca; acc[i].z *= ca; acc[i].w *= ca;
                #pragma unroll
                for (int q = 0; q < 4; q++) {
                    const float cb = ex2_fast(mj[q][i] - ref);
                    l[i] = fmaf(lj[q][i], cb, l[i]);
                    acc[i].x = fmaf(v[q][i].x, cb, acc[i].x); acc[i].y = fmaf(v[q][i].y, cb, acc[i].y);
                    acc[i].z = fmaf(v[q][i].z, cb, acc[i].z); acc[i].w = fmaf(v[q][i].w, cb, acc[i].w);
                }
            }
        }
    }
};

template <int HS_, int ROWS, int PJ_WARPS>
__global__ void __launch_bounds__(PJ_WARPS * 32)
paged_few_join_kernel(const FewArgs a, int shares, int G, int hs) {
    constexpr int R = ROWS / 4;
    __shared__ float4 merged[PJ_WARPS][ROWS][PJ_CHANNELS / 4];
    __shared__ float ms[PJ_WARPS][ROWS], ls[PJ_WARPS][ROWS];
    __shared__ PagedJoin joins[PJ_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, k0 = blockIdx.x * PJ_WARPS;
    pdl_wait();                                                // the partials
    pdl_trigger();
    if (threadIdx.x < PJ_WARPS * 8) {
        const int k = k0 + threadIdx.x / 8;
        reinterpret_cast<int*>(joins)[threadIdx.x] = k < shares ? reinterpret_cast<const int*>(a.ws)[k * 8 + threadIdx.x % 8] : 0;
    }
    __syncthreads();
    const float* base = few_parts(a.ws, shares);
    const int ch0 = blockIdx.y * PJ_CHANNELS;
    auto store = [&](const PagedJoin& jn, int r, int c4, float4 o, float m, float l) {
        const float inv = paged_inverse(m, l);
        const int row = jn.row + r, token = row / G;
        if (ch0 + c4 * 4 < hs)
            *reinterpret_cast<uint2*>(a.out + (jn.first + token) * a.ldo + (jn.g * G + row - token * G) * hs + ch0 + c4 * 4) =
                make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
    };
    FewSum<ROWS> sum;
    const int mine = joins[warp].parts;
    if (mine > 0 && mine <= PJ_ALONE) {
        const int rows = min(ROWS, joins[warp].count * G - joins[warp].row);
        sum.template add<HS_>(base, k0 + warp, mine, rows, 0, 1, ch0 + (lane & 7) * 4);
        #pragma unroll
        for (int i = 0; i < R; i++) if ((lane >> 3) + 4 * i < rows) store(joins[warp], (lane >> 3) + 4 * i, lane & 7, sum.acc[i], sum.m[i], sum.l[i]);
    }
    for (int i = 0; i < PJ_WARPS; i++) {
        const int parts = joins[i].parts;                      // (the same for all warps)
        if (parts <= PJ_ALONE) continue;
        const int rows = min(ROWS, joins[i].count * G - joins[i].row);
        sum.template add<HS_>(base, k0 + i, parts, rows, warp, PJ_WARPS, ch0 + (lane & 7) * 4);
        #pragma unroll
        for (int e = 0; e < R; e++) {
            const int r = (lane >> 3) + 4 * e;
            merged[warp][r][lane & 7] = sum.acc[e];
            if ((lane & 7) == 0) { ms[warp][r] = sum.m[e]; ls[warp][r] = sum.l[e]; }
        }
        __syncthreads();
        const int r = threadIdx.x / (PJ_CHANNELS / 4), c4 = threadIdx.x % (PJ_CHANNELS / 4);
        if (r < rows) {
            float mn = -INFINITY;
            #pragma unroll
            for (int w = 0; w < PJ_WARPS; w++) mn = fmaxf(mn, ms[w][r]);
            const float ref = mn == -INFINITY ? 0.f : mn;
            float l = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            #pragma unroll
            for (int w = 0; w < PJ_WARPS; w++) {
                const float cw = ex2_fast(ms[w][r] - ref);
                const float4 x = merged[w][r][c4];
                l = fmaf(ls[w][r], cw, l);
                o.x = fmaf(x.x, cw, o.x); o.y = fmaf(x.y, cw, o.y); o.z = fmaf(x.z, cw, o.z); o.w = fmaf(x.w, cw, o.w);
            }
            store(joins[i], r, c4, o, mn, l);
        }
        __syncthreads();                                       // the next one is merged in the same place
    }
}

// How a call is cut, from what the host knows: rows of a group, warps that take a piece together, keys of a unit, units that a piece counts besides, blocks; whether parts are joined
struct FewPlan {
    int rows, coop, unit_log2, over, blocks;
    bool joins;
    long long units;
    int shares() const { return blocks * (PF_WARPS / coop); }
};
FewPlan few_plan(const PagedCache* c, int N, int NH) {
    int sms = llmc_device_sm_count(); if (sms <= 0) sms = 148;
    const long long keys = (long long)c->table_width << c->page_shift;
    FewPlan p;
    p.rows = (long long)N * (NH / c->heads) > 8LL * c->sequences ? 16 : 8;
    const long long pieces = paged_few_pieces(c, N, NH, p.rows);
    // Pieces of at most 256 keys are not cut: one of 161 keys takes 6 us, cut and joined 12.  Fewer pieces than SMs are cut by blocks whose four warps share the keys, more of them by warps, which
    // do not wait for one another but leave more parts to be joined (us, blocks / warps: 8 pieces of 2000 keys 9.1 / 15.9, of 20000 22.7 / 31, 32 of 48 rows in all 13.9 / 18.9; heads of 64: 864 of up
    // to 1000 keys 33.9 / 29.6).  Groups of 8 rows of wide heads are best cut by blocks up to some more (256 of up to 8192 104.4 / 106.3, 768 of up to 1000 34.3 / 35.9, 1536 of up to 500 35.9 / 35.5;
    // groups of 16 rows: 400 of up to 4000 67.3 / 64.3).
    p.joins = keys > 256;
    p.coop = pieces <= (p.rows == 8 && c->hs > 64 ? 6 : 1) * sms ? 4 : 1;
    p.unit_log2 = !p.joins ? 8 : p.coop == 4 ? 6 : 4;          // a tile of each warp
    // What it takes to begin and to end a piece, in units of a share.  (Counted as nothing, shares of many short pieces end late: 1024 pieces of up to 500 keys 45 us, as one unit 36.5, two 35.4,
    // four 36; 512 of up to 1000 29.7, 26.3, 25, 24.9.)
    p.over = !p.joins ? 0 : p.coop == 4 ? 1 : 2;
    p.units = pieces * (p.over + CEIL_DIV(keys > 0 ? keys : 1, 1LL << p.unit_log2));
    const int teams = PF_WARPS / p.coop;
    p.blocks = (int)(p.units < 2LL * sms * teams ? (p.units + teams - 1) / teams : 2 * sms);
    return p;
}

template <int HS_, int ROWS, int COOP>
int few_launch(const PagedCache* c, const FewArgs& a, const FewPlan& p, cudaStream_t stream) {
    constexpr int smem = pf_smem_bytes<HS_, COOP>();
    static bool done[64];
    int rc = paged_shared_memory(paged_few_kernel<HS_, ROWS, COOP>, smem, done);
    if (rc) return rc;
    CUtensorMap tmK, tmV;
    if ((rc = paged_maps(&tmK, &tmV, c, a.layer, a.box))) return rc;
    CUDA_CHECK(launch_pdl(paged_few_kernel<HS_, ROWS, COOP>, dim3(p.blocks), dim3(PF_THREADS), smem, stream, 0, tmK, tmV, *c, a));
    constexpr int W = COOP == 1 ? 4 : 8;
    if (p.joins && p.shares() > 1)
        CUDA_CHECK(launch_pdl(paged_few_join_kernel<HS_, ROWS, W>, dim3(CEIL_DIV(p.shares(), W), CEIL_DIV(c->hs, PJ_CHANNELS)), dim3(W * 32), 0, stream, 0, a, p.shares(), a.NH / c->heads,
                              c->hs));
    return 0;
}
template <int HS_>
int few_dispatch(const PagedCache* c, const FewArgs& a, const FewPlan& p, cudaStream_t stream) {
    if (p.rows == 8) return p.coop == 4 ? few_launch<HS_, 8, 4>(c, a, p, stream) : few_launch<HS_, 8, 1>(c, a, p, stream);
    return p.coop == 4 ? few_launch<HS_, 16, 4>(c, a, p, stream) : few_launch<HS_, 16, 1>(c, a, p, stream);
}

}  // namespace

int paged_maps(CUtensorMap* tmK, CUtensorMap* tmV, const PagedCache* c, int layer, int box_rows) {
    for (int kv = 0; kv < 2; kv++) {
        const bf16* base = kv ? c->v + layer * c->v_layer : c->k + layer * c->k_layer;
        const uint64_t dims[4] = {(uint64_t)c->hs, (uint64_t)c->heads, 1ull << c->page_shift, (uint64_t)c->pages};
        const uint64_t strides[4] = {2, 2ull * (kv ? c->v_head : c->k_head), 2ull * (kv ? c->v_row : c->k_row), 2ull * (kv ? c->v_page : c->k_page)};
        const uint32_t box[4] = {64, 1, (uint32_t)box_rows, 1};
        const int rc = llmc_get_tensormap(kv ? tmV : tmK, base, 2, 4, dims, strides, box, 3 | TENSORMAP_L2_128B);
        if (rc) return rc;
    }
    return 0;
}

bool paged_few_fits(const PagedCache* c, int N, int NH) { return few_plan(c, N, NH).units < PAGED_UNITS && (long long)N * (NH / c->heads) < PAGED_UNITS; }

// fp32 words of workspace that llmc_paged_attention needs for a batch of N rows
extern "C" long long llmc_paged_attention_workspace(const PagedCache* c, int N, int NH) {
    if (paged_wide(c, N, NH)) return paged_wide_workspace(c, N, NH);
    const FewPlan p = few_plan(c, N, NH);
    return (long long)p.shares() * ((int)sizeof(PagedJoin) / 4 + (p.joins ? 2 * p.rows * (2 + (c->hs > 64 ? 128 : 64)) : 0));
}

// Launches of such a call
extern "C" int llmc_paged_attention_launches(const PagedCache* c, int N, int NH) {
    if (paged_wide(c, N, NH)) return paged_wide_launches(c, N, NH);
    const FewPlan p = few_plan(c, N, NH);
    return p.joins && p.shares() > 1 ? 2 : 1;
}

// Arguments in 64-bit words (paged.cuh).  Work that does not fit 32-bit counts (2^30 units of 16 to 128 keys, each sequence counted with all keys that the table has room for) is refused: -7; more
// than 2^30 rows, as by llmc_paged_rope_cache: -1
extern "C" int llmc_paged_attention(const PagedAttentionCall* call) {
    const PagedCache* c = call->cache;
    if (call->N <= 0 || call->N > 1 << 30 || call->NH <= 0 || call->NH > 0x7fffffff) return -1;
    const int N = (int)call->N, NH = (int)call->NH, layer = (int)call->layer;
    const long long ldo = call->ldo, ldq = call->ldq;
    bf16* out = call->out;
    const bf16* q = call->q;
    const long long* tree = call->tree;
    float* ws = call->ws;
    cudaStream_t stream = call->stream;
    if (c->sequences <= 0 || c->pages <= 0 || NH % c->heads || layer < 0 || layer >= c->layers || c->hs > 128 || c->hs % 8 || c->page_shift < 3 || ldq % 8 || ldo % 8) return -1;
    if (paged_wide(c, N, NH)) return paged_wide_launch(c, {out, ws, q, tree, ldo, ldq, N, NH, layer, llmc_status_ptr()}, stream);
    const FewPlan p = few_plan(c, N, NH);
    if (!paged_few_fits(c, N, NH)) return -7;
    const FewArgs a = {{out, ws, q, tree, ldo, ldq, N, NH, layer, llmc_status_ptr()}, p.unit_log2, p.over, c->page_shift == 3 ? 8 : 16, 1.0f / sqrtf((float)c->hs) * PF_LOG2E};
    return c->hs > 64 ? few_dispatch<128>(c, a, p, stream) : few_dispatch<64>(c, a, p, stream);
}
