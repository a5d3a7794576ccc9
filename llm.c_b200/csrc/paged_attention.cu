// Attention of ragged new tokens over a key / value cache in pages (paged.cuh):
//
//   out[n, h] = sum over the keys s that row n sees of softmax_s(q[n, h] . K[s, g] / sqrt(HS)) V[s, g],  g = h / (NH / NKV); 0 where it sees none.
//   Token i of a sequence of `len` keys with `count` new ones sees slots 0 .. len - count + i; with `tree` it sees slots below len - count, and slot len - count + j
//   where bit j of tree[n] is set (at most 64 new tokens of a sequence).
//
// Few rows to a cached head (a decoding step): reading the cache once is all the work there is.  A piece is one cached head of one sequence for 8 query rows (its tokens' grouped heads).
//   * Each of a block's 4 warps walks tiles of 16 keys whose K and V rows arrive by cp.async through a ring of its own (16-byte chunks of row j XOR-swizzled by j & 7); the next 32 tiles'
//     pages are looked up at once, a lane for each, so that no load waits for the table.
//   * S = Q K^T and O += P V on warp-level MMAs, the query rows as the 16-row operand (8 of them used).  P keeps 16 bits: the upper 8 as a bf16 in rows 0..7 of the operand, the next 8 in
//     rows 8..15, which are idle otherwise; the two halves of the accumulator are added at the end.  (One bf16 would leave an error as large as the output's rounding.)
//   * Slots behind the length are not read: their rows in shared memory are zeros, whatever the page holds.
//   * Running (max, sum, accumulator) per warp, merged over the warps through shared memory; partials of pieces that a share ends in go to a workspace in fp32.
#include "paged_attention_ops.h"
#include "pdl.cuh"

namespace {

constexpr int PF_WARPS = 4;
constexpr int PF_THREADS = PF_WARPS * 32;
constexpr int PF_ROWS = 8;            // query rows of a piece
constexpr int PF_TILE = 16;           // keys per tile of a warp
constexpr int PF_TRIP = PF_WARPS * PF_TILE;
constexpr int PF_STAGES = 3;
constexpr float PF_LOG2E = 1.4426950408889634f;

DEVINL void cp_async16_or_zero(void* smem_dst, const void* gsrc, bool in) {     // gsrc is a readable address either way
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem_dst)), "l"(gsrc), "r"(in ? 16 : 0) : "memory");
}
DEVINL void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> DEVINL void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
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

// The workspace holds two partials per block: PF_ROWS x (HS_ + 2) words each
struct FewArgs : PagedAttention {
    int unit;                  // keys of a unit, a multiple of PF_TRIP
    float scale_log2e;
};

template <int HS_> __host__ __device__ constexpr int pf_part_floats() { return PF_ROWS * (HS_ + 2); }
template <int HS_> __host__ __device__ constexpr int pf_ring_bytes() { return PF_STAGES * 2 * PF_TILE * HS_ * 2; }      // of one warp
template <int HS_> __host__ __device__ constexpr int pf_smem_bytes() {
    return PF_WARPS * (pf_ring_bytes<HS_>() > pf_part_floats<HS_>() * 4 ? pf_ring_bytes<HS_>() : pf_part_floats<HS_>() * 4);
}

struct FewUnits {
    const PagedCache& c;
    const FewArgs& a;
    int G;
    DEVINL int groups(const PagedSpan& s) const { return (int)(((long long)s.count * G + PF_ROWS - 1) / PF_ROWS); }
    DEVINL int tiles(const PagedSpan& s) const { return s.keys > 0 ? (s.keys + a.unit - 1) / a.unit : 1; }
    DEVINL long long operator()(int b) const {
        const PagedSpan s = paged_span(c, b, a.N, a.status, 0x48);
        return (long long)groups(s) * c.heads * tiles(s);
    }
};

// Writes rows of a merged result: row r of group `grp` is token r / G, head g * G + r % G
DEVINL bf16* few_out(const FewArgs& a, const PagedSpan& s, int G, int g, int row, int hs) {
    return a.out + (s.first + row / G) * a.ldo + (g * G + row % G) * hs;
}

template <int HS_>
__global__ void __launch_bounds__(PF_THREADS)
paged_few_kernel(const PagedCache c, const FewArgs a) {
    pdl_wait();
    pdl_trigger();
    constexpr int ROWB = HS_ * 2;              // bytes of a key row
    constexpr int CHUNKS = HS_ / 8;            // 16-byte chunks of a row
    constexpr int KS = HS_ / 16;               // 16-channel steps
    constexpr int STAGE = 2 * PF_TILE * ROWB;  // K tile, V tile
    constexpr int PART = pf_part_floats<HS_>();
    extern __shared__ __align__(16) uint8_t pf_smem[];
    __shared__ long long red[PF_WARPS + 2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int gq = lane >> 2, tq4 = lane & 3;                  // MMA fragment coordinates: row gq, column pair tq4
    uint8_t* ring = pf_smem + warp * pf_ring_bytes<HS_>();
    const int hs = c.hs, G = a.NH / c.heads;
    const FewUnits units{c, a, G};
    long long before;
    int b0, b1;
    const long long total = paged_total<PF_THREADS>(c.sequences, units, red, before, b0, b1);
    const int blocks = (int)min((long long)gridDim.x, total);  // with a share
    if ((int)blockIdx.x >= blocks) return;
    const long long first = paged_share(total, blockIdx.x, blocks), end = paged_share(total, blockIdx.x + 1, blocks);
    paged_locate(first, before, b0, b1, units, red + PF_WARPS);
    __syncthreads();
    int b = (int)red[PF_WARPS];
    long long at = red[PF_WARPS + 1];                          // units in front of sequence b
    const int in_page = (1 << c.page_shift) - 1;

    for (long long u = first; u < end;) {
        PagedSpan s = paged_span(c, b, a.N, a.status, 0x48);
        long long mine = (long long)units.groups(s) * c.heads * units.tiles(s);
        while (u >= at + mine) {                               // (uniform; ends, since u < total)
            at += mine;
            b++;
            s = paged_span(c, b, a.N, a.status, 0x48);
            mine = (long long)units.groups(s) * c.heads * units.tiles(s);
        }
        const int nt = units.tiles(s), ng = units.groups(s);
        const int piece = (int)((u - at) / nt), t0 = (int)((u - at) - (long long)piece * nt), t1 = (int)min((long long)nt, t0 + (end - u));
        const int g = piece / ng, grp = piece - g * ng;
        u += t1 - t0;
        const int rows = min(PF_ROWS, s.count * G - grp * PF_ROWS);
        const int context = s.keys - s.count;
        const bool too_many = a.tree && s.count > 64;
        if (too_many && threadIdx.x == 0) record_error(a.status, ST_BAD_ARG, 0x49);
        const int k0 = t0 * a.unit, k1 = too_many ? k0 : min(s.keys, t1 * a.unit);
        const bf16 *kbase = c.k + a.layer * c.k_layer + g * c.k_head, *vbase = c.v + a.layer * c.v_layer + g * c.v_head;
        const int kt0 = k0 + warp * PF_TILE;

        // pages of the warp's next 32 tiles, a lane for each; of 8-row pages a tile has two
        int look = kt0 - 32 * PF_TRIP, page_lo = -1, page_hi = -1;
        auto fetch = [&](int kt, int st) {
            if (kt < k1) {
                if (kt >= look + 32 * PF_TRIP) {
                    look = kt;
                    const int slot = kt + lane * PF_TRIP;
                    page_lo = slot < k1 ? paged_page(c, b, slot, a.status, 0x4A) : -1;
                    page_hi = c.page_shift == 3 && slot + 8 < k1 ? paged_page(c, b, slot + 8, a.status, 0x4A) : page_lo;
                }
                const int from = (kt - look) / PF_TRIP;
                const int p0 = __shfl_sync(0xffffffffu, page_lo, from), p1 = __shfl_sync(0xffffffffu, page_hi, from);
                uint8_t* dst = ring + st * STAGE;
                #pragma unroll
                for (int i = 0; i < PF_TILE * CHUNKS / 32; i++) {
                    const int id = i * 32 + lane, row = id / CHUNKS, ch = id % CHUNKS, slot = kt + row;
                    const int page = row < 8 ? p0 : p1;
                    const bool in = slot < k1 && page >= 0 && ch * 8 < hs;
                    const long long r = in ? slot & in_page : 0, p = in ? page : 0, x = in ? ch * 8 : 0;
                    const int off = row * ROWB + ((ch ^ (row & 7)) * 16);
                    cp_async16_or_zero(dst + off, kbase + p * c.k_page + r * c.k_row + x, in);
                    cp_async16_or_zero(dst + PF_TILE * ROWB + off, vbase + p * c.v_page + r * c.v_row + x, in);
                }
            }
            cp_async_commit();                                 // possibly empty: the group count per tile stays one
        };
        #pragma unroll
        for (int st = 0; st < PF_STAGES - 1; st++) fetch(kt0 + st * PF_TRIP, st);

        // query rows; the A operand of S: lane holds channels 2 tq4, 2 tq4 + 1 and + 8, + 9 of row gq.  Rows past `rows` are zero and dropped at the end.
        uint32_t qa[KS][2];
        const int qrow = grp * PF_ROWS + (gq < rows ? gq : 0), token = qrow / G;
        {
            const bf16* qr = a.q + (s.first + token) * a.ldq + (g * G + qrow % G) * hs + 2 * tq4;
            #pragma unroll
            for (int kk = 0; kk < KS; kk++) {
                qa[kk][0] = gq < rows && kk * 16 < hs ? *reinterpret_cast<const uint32_t*>(qr + kk * 16) : 0u;
                qa[kk][1] = gq < rows && kk * 16 + 8 < hs ? *reinterpret_cast<const uint32_t*>(qr + kk * 16 + 8) : 0u;
            }
        }
        const unsigned long long bits = a.tree ? (unsigned long long)a.tree[s.first + token] : 0;
        const int limit = min(k1, a.tree ? context : context + token + 1);        // keys [0, limit) are visible to this lane's row; with a tree, others behind them
        const float sl2 = a.scale_log2e;
        float m = -INFINITY, l = 0.f;                          // of row gq; l: this lane's keys only
        float acc[HS_ / 8][4];                                 // columns 2 tq4, + 1 of channel group n: [0,1] from the upper bits of P, [2,3] from the lower
        #pragma unroll
        for (int n = 0; n < HS_ / 8; n++) { acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f; }
        const int mrow = lane & 7, mid = lane >> 3;            // ldmatrix: lane supplies the row address of matrix lane / 8, row lane % 8
        int st = 0;
        for (int kt = kt0; kt < k1; kt += PF_TRIP) {
            fetch(kt + (PF_STAGES - 1) * PF_TRIP, st == 0 ? PF_STAGES - 1 : st - 1);
            cp_async_wait<PF_STAGES - 1>();
            __syncwarp();
            const uint32_t kb = smem_u32(ring + st * STAGE), vb = kb + PF_TILE * ROWB;
            // ---- S (row gq, keys 2 tq4 + {0,1} of each group of 8 keys)
            float sc[2][4];
            #pragma unroll
            for (int h = 0; h < 2; h++) { sc[h][0] = sc[h][1] = sc[h][2] = sc[h][3] = 0.f; }
            #pragma unroll
            for (int kk = 0; kk < KS; kk++) {
                uint32_t kf[4];     // matrices: keys 0-7 channels 0-7 / 8-15 of the step, keys 8-15 likewise
                const int row = (mid >> 1) * 8 + mrow, ch = kk * 2 + (mid & 1);
                ldmatrix4(kf, kb + row * ROWB + ((ch ^ (row & 7)) * 16));
                mma_16x8x16(sc[0], qa[kk][0], 0u, qa[kk][1], 0u, kf[0], kf[1]);
                mma_16x8x16(sc[1], qa[kk][0], 0u, qa[kk][1], 0u, kf[2], kf[3]);
            }
            // ---- running softmax of row gq (base 2); the four lanes of a row hold its 16 keys
            float sv[4];
            #pragma unroll
            for (int e = 0; e < 4; e++) {
                const int key = kt + (e >> 1) * 8 + 2 * tq4 + (e & 1);
                bool seen = key < limit;
                if (a.tree && key >= context) seen = key < k1 && (bits >> (key - context) & 1);
                sv[e] = seen ? sc[e >> 1][e & 1] * sl2 : -INFINITY;
            }
            float mn = fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3]));
            mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 1));
            mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 2));
            mn = fmaxf(mn, m);
            const float mref = mn == -INFINITY ? 0.f : mn;     // no key seen yet: every probability below is 2^-inf = 0
            const float corr = ex2_fast(m - mref);
            float p[4];
            #pragma unroll
            for (int e = 0; e < 4; e++) p[e] = ex2_fast(sv[e] - mref);
            l = l * corr + ((p[0] + p[1]) + (p[2] + p[3]));
            m = mn;
            if (__any_sync(0xffffffffu, corr != 1.0f)) {
                #pragma unroll
                for (int n = 0; n < HS_ / 8; n++) { acc[n][0] *= corr; acc[n][1] *= corr; acc[n][2] *= corr; acc[n][3] *= corr; }
            }
            uint32_t hi[2], lo[2];
            #pragma unroll
            for (int h = 0; h < 2; h++) {
                hi[h] = top_bf16x2(p[2 * h], p[2 * h + 1]);
                const float2 hf = unpack_bf16x2(hi[h]);
                lo[h] = pack_bf16x2(p[2 * h] - hf.x, p[2 * h + 1] - hf.y);
            }
            // ---- O += P V: 16 keys, 16 channels per ldmatrix
            #pragma unroll
            for (int n2 = 0; n2 < HS_ / 16; n2++) {
                uint32_t vf[4];     // matrices: keys 0-7 / 8-15 of channels 0-7 of the pair of groups, then of channels 8-15
                const int row = (mid & 1) * 8 + mrow, ch = n2 * 2 + (mid >> 1);
                ldmatrix4_trans(vf, vb + row * ROWB + ((ch ^ (row & 7)) * 16));
                mma_16x8x16(acc[2 * n2], hi[0], lo[0], hi[1], lo[1], vf[0], vf[1]);
                mma_16x8x16(acc[2 * n2 + 1], hi[0], lo[0], hi[1], lo[1], vf[2], vf[3]);
            }
            __syncwarp();                                      // the stage may be refilled
            st = st + 1 == PF_STAGES ? 0 : st + 1;
        }
        cp_async_wait<0>();
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        // ---- merge the warps in warp order (the rings are free now)
        __syncthreads();
        float* wp = reinterpret_cast<float*>(pf_smem) + warp * PART;
        #pragma unroll
        for (int n = 0; n < HS_ / 8; n++)
            *reinterpret_cast<float2*>(wp + gq * HS_ + n * 8 + 2 * tq4) = make_float2(acc[n][0] + acc[n][2], acc[n][1] + acc[n][3]);
        if (tq4 == 0) { wp[PF_ROWS * HS_ + gq] = m; wp[PF_ROWS * HS_ + PF_ROWS + gq] = l; }
        __syncthreads();
        const float* w0 = reinterpret_cast<const float*>(pf_smem);
        const bool whole = t0 == 0 && t1 == nt;
        float* part = a.ws + (size_t)(2 * blockIdx.x + (t0 == 0)) * PART;
        for (int i = threadIdx.x; i < rows * (HS_ / 2); i += PF_THREADS) {
            const int r = i / (HS_ / 2), ch = (i - r * (HS_ / 2)) * 2;
            float mn = -INFINITY;
            #pragma unroll
            for (int w = 0; w < PF_WARPS; w++) mn = fmaxf(mn, w0[w * PART + PF_ROWS * HS_ + r]);
            float x = 0.f, y = 0.f, ls = 0.f;
            #pragma unroll
            for (int w = 0; w < PF_WARPS; w++) {
                const float mw = w0[w * PART + PF_ROWS * HS_ + r];
                const float cw = (mw == -INFINITY) ? 0.f : ex2_fast(mw - mn);
                const float2 v = *reinterpret_cast<const float2*>(w0 + w * PART + r * HS_ + ch);
                x += v.x * cw;
                y += v.y * cw;
                ls += w0[w * PART + PF_ROWS * HS_ + PF_ROWS + r] * cw;
            }
            if (whole) {
                const float inv = ls == 0.f ? 0.f : 1.0f / ls;
                if (ch < hs) *reinterpret_cast<uint32_t*>(few_out(a, s, G, g, grp * PF_ROWS + r, hs) + ch) = pack_bf16x2(x * inv, y * inv);
            } else {
                *reinterpret_cast<float2*>(part + r * HS_ + ch) = make_float2(x, y);
                if (ch == 0) { part[PF_ROWS * HS_ + r] = mn; part[PF_ROWS * HS_ + PF_ROWS + r] = ls; }
            }
        }
        __syncthreads();                                       // the rings belong to the next piece
    }
}

// Joins the partials of a piece that lies in several shares: the block of the first share that begins inside it does, for a slice of its rows and channels
template <int HS_>
__global__ void __launch_bounds__(PF_THREADS)
paged_few_join_kernel(const PagedCache c, const FewArgs a, int most_blocks) {
    __shared__ long long red[PF_WARPS + 2];
    constexpr int PART = pf_part_floats<HS_>();
    const int k = blockIdx.x + 1, G = a.NH / c.heads, hs = c.hs;
    const FewUnits units{c, a, G};
    long long before;
    int b0, b1;
    const long long total = paged_total<PF_THREADS>(c.sequences, units, red, before, b0, b1);
    const int blocks = (int)min((long long)most_blocks, total);
    if (k >= blocks) { pdl_wait(); pdl_trigger(); return; }
    const long long u = paged_share(total, k, blocks);
    paged_locate(u, before, b0, b1, units, red + PF_WARPS);
    __syncthreads();
    const int b = (int)red[PF_WARPS];
    const long long at = red[PF_WARPS + 1];
    const PagedSpan s = paged_span(c, b, a.N, a.status, 0x48);
    const int nt = units.tiles(s), ng = units.groups(s);
    const int piece = (int)((u - at) / nt);
    const long long s0 = at + (long long)piece * nt, s1 = s0 + nt;
    const int g = piece / ng, grp = piece - g * ng, rows = min(PF_ROWS, s.count * G - grp * PF_ROWS);
    pdl_wait();                                                // the partials
    pdl_trigger();
    if (u == s0 || paged_share(total, k - 1, blocks) > s0) return;             // not inside a piece, or not the first share that begins there
    int last = k;
    while (last + 1 < blocks && paged_share(total, last + 1, blocks) < s1) last++;
    const float* p0 = a.ws + (size_t)(2 * k - 1) * PART;          // of block k - 1
    for (int i = threadIdx.x; i < rows * (HS_ / 2); i += PF_THREADS) {
        const int r = i / (HS_ / 2), ch = (i - r * (HS_ / 2)) * 2;
        if (ch >= hs) continue;
        float m = p0[PF_ROWS * HS_ + r], l = p0[PF_ROWS * HS_ + PF_ROWS + r];
        float2 v = *reinterpret_cast<const float2*>(p0 + r * HS_ + ch);
        float x = v.x, y = v.y;
        for (int j = k; j <= last; j++) {
            const float* p = a.ws + (size_t)(2 * j) * PART;
            const float mj = p[PF_ROWS * HS_ + r], mn = fmaxf(m, mj), ref = mn == -INFINITY ? 0.f : mn;
            const float ca = ex2_fast(m - ref), cb = ex2_fast(mj - ref);
            v = *reinterpret_cast<const float2*>(p + r * HS_ + ch);
            x = x * ca + v.x * cb;
            y = y * ca + v.y * cb;
            l = l * ca + p[PF_ROWS * HS_ + PF_ROWS + r] * cb;
            m = mn;
        }
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        *reinterpret_cast<uint32_t*>(few_out(a, s, G, g, grp * PF_ROWS + r, hs) + ch) = pack_bf16x2(x * inv, y * inv);
    }
}

// Blocks and keys of a unit.  `most`: a bound of the number of pieces; keys: what the table can hold
struct FewPlan { int blocks, unit; };
FewPlan few_plan(const PagedCache* c, int N, int NH) {
    int sms = llmc_device_sm_count(); if (sms <= 0) sms = 148;
    const int G = NH / c->heads;
    const long long keys = (long long)c->table_width << c->page_shift;
    const long long pieces = ((long long)N * G / PF_ROWS + c->sequences) * c->heads;
    FewPlan p;
    p.unit = keys <= 4 * PF_TRIP ? 4 * PF_TRIP : PF_TRIP;
    const long long units = pieces * CEIL_DIV(keys > 0 ? keys : 1, p.unit);
    p.blocks = (int)(units < 2 * sms ? units : 2 * sms);
    return p;
}

template <int HS_>
int few_launch(const PagedCache* c, const FewArgs& a, const FewPlan& p, cudaStream_t stream) {
    constexpr int smem = pf_smem_bytes<HS_>();
    static bool done[64];
    const int rc = paged_shared_memory(paged_few_kernel<HS_>, smem, done);
    if (rc) return rc;
    CUDA_CHECK(launch_pdl(paged_few_kernel<HS_>, dim3(p.blocks), dim3(PF_THREADS), smem, stream, 0, *c, a));
    if (((long long)c->table_width << c->page_shift) > p.unit && p.blocks > 1)
        CUDA_CHECK(launch_pdl(paged_few_join_kernel<HS_>, dim3(p.blocks - 1), dim3(PF_THREADS), 0, stream, 0, *c, a, p.blocks));
    return 0;
}

}  // namespace

// fp32 words of workspace that llmc_paged_attention needs for a batch of N rows
extern "C" long long llmc_paged_attention_workspace(const PagedCache* c, int N, int NH) {
    if (paged_wide(c, N, NH)) return paged_wide_workspace(c, N, NH);
    return 2LL * few_plan(c, N, NH).blocks * (c->hs > 64 ? pf_part_floats<128>() : pf_part_floats<64>());
}

extern "C" int llmc_paged_attention(bf16* out, const PagedCache* c, const bf16* q, const long long* tree, float* ws, int N, long long ldo, long long ldq, int NH, int layer, cudaStream_t stream) {
    if (N <= 0 || c->sequences <= 0 || NH <= 0 || NH % c->heads || layer < 0 || layer >= c->layers || c->hs > 128 || c->hs % 8 || ldq % 8 || ldo % 8) return -1;
    if (paged_wide(c, N, NH)) return paged_wide_launch(c, {out, ws, q, tree, ldo, ldq, N, NH, layer, llmc_status_ptr()}, stream);
    const FewPlan p = few_plan(c, N, NH);
    const FewArgs a = {{out, ws, q, tree, ldo, ldq, N, NH, layer, llmc_status_ptr()}, p.unit, 1.0f / sqrtf((float)c->hs) * PF_LOG2E};
    return c->hs > 64 ? few_launch<128>(c, a, p, stream) : few_launch<64>(c, a, p, stream);
}
