// Attention of portions of prompts over a cache held in 4 bits (int4.cuh) on the 5th-generation tensor cores, bfloat16 queries: S = Q K^T and
// O += P V are tcgen05.mma instructions (float16 operands, float32 sums in tensor memory).
//
// A block takes up to 256 rows - tokens by the heads that share a KV head, of a tile of 64 tokens - as two products of 128 rows, and all keys
// they see, 64 at a time.  Six warps bring the keys' and values' codes in from the pages (bulk copies, three tiles of 16 keys a warp on the way)
// and write them, as float16 values, into the operands' shared tiles; a thread for each 128 rows issues their products; eight warps hold a row a
// thread for the softmax.  Values of 64 keys serve 256 rows, so that the work of making them (14 instructions for 8 values) stays below the
// softmax's (some 7 for a score).
// Tensor memory holds two tiles of scores for each 128 rows and their outputs.  A tile's probabilities take the place of its scores, as the
// first operand of P V: the products of tile j + 1's scores run while tile j's softmax does, and neither waits for P V of the tile before.  (With
// one tile of scores, P in shared memory and one issuing thread, a tile of 64 keys took 2.27 us, of which 1.3 were hand-overs that stayed
// with all work left out.)
//
// 1,733 tokens after 6,000, 32 heads over 8 of 128: 294 us, 0.40 of the arithmetic peak: a tile of 64 keys takes some 2,500 cycles, of which the
// exponentials of 256 rows take 1,024, the products 1,300, and the softmax's chain (scores there, 1,550 cycles of arithmetic, probabilities
// stored, products issued) is the longest; 224 blocks for 148 SMs take one and a half rounds.
//
// Roundings: c s + z to float16 once (by 2^-11 of itself at most; the codes are exact); a query row brought into [2^14, 2^15) by a power of two is exact in
// float16 down to 2^-30 of its largest; a probability is kept as 2^(S - m) with m six below the running maximum, so that float16 holds it to
// 2^-11 of itself down to 2^-20 of the largest.  A group of values that is not a number is put into the tile as zeros and reaches the rows that
// see its key at the end.
//
// Keys' and values' channels lie in the order in which codes come out of their words; the queries' channels are laid out to match, and
// the outputs' are put back where they are stored.
//
// Every wait on an mbarrier is bounded; on a timeout the block sets a status of 61 to 68, waits (with the same limit) for its copies and products
// that are under way, frees its tensor memory and returns.  Tensor memory is
// taken behind the wait for the kernels in front and before the kernels behind may start: a neighbour that waits for this grid never holds
// what this grid waits for.
#include "int4.cuh"
#include "int4_ring.h"

namespace {

constexpr int BN = 64, STAGES = 3, RAW = 3;      // RAW: tiles of codes a making warp has on the way
constexpr int MAKERS = 6, SOFTMAX = 8, THREADS = 32 * (2 + MAKERS + SOFTMAX);
constexpr float LIFT = 6.0f, HEADROOM = 8.0f;
// From this magnitude of the reference on, float32's steps (1 and more) tell in what a probability comes out as: there, they are cut to the LIFT and
// HEADROOM that they may have (the reference is rounded down: none is lost).
constexpr float COARSE = 0x1p23f;

struct Args {
    const __nv_bfloat16* q;        // [T, heads, d]: token stride q_stride, heads d apart
    __nv_bfloat16* out;
    const unsigned char* pages;
    const int *seq_slot, *q_start, *ctx_len, *block_table, *tiles;
    int* status;
    long long q_stride;
    int nh, nkv, page_size, max_pages, num_pages, window, block_rows;
    float scale_log2;
};

__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(i4_smem(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(i4_smem(bar)) : "memory");
}
// Shared-memory operand descriptors, 128-byte swizzle.  K-major: rows of 128 bytes along K, 8-row groups 1024 bytes apart.  MN-major: rows of 128
// bytes along MN (64 elements), one row per k, 8-row groups 1024 bytes apart, the next 64 MN elements ``next`` bytes further.
__device__ __forceinline__ uint64_t desc_kmajor(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ uint64_t desc_mnmajor(uint32_t addr, uint32_t next) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)(next >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// One lane of a whole warp issues (always the same one): descriptors stay in registers that a warp shares.
__device__ __forceinline__ void umma(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n.reg .pred p, q;\nelect.sync _|q, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\n@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
                 ::"r"(d_tmem), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
// the same with the first operand in tensor memory
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n.reg .pred p, q;\nelect.sync _|q, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\n@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
                 ::"r"(d_tmem), "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("{\n.reg .pred q;\nelect.sync _|q, 0xffffffff;\n@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}"
                 ::"r"(i4_smem(bar)) : "memory");
}
__device__ __forceinline__ void tmem_ld32_issue(uint32_t taddr, uint32_t* q) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]), "=r"(q[4]), "=r"(q[5]), "=r"(q[6]), "=r"(q[7]),
                   "=r"(q[8]), "=r"(q[9]), "=r"(q[10]), "=r"(q[11]), "=r"(q[12]), "=r"(q[13]), "=r"(q[14]), "=r"(q[15]),
                   "=r"(q[16]), "=r"(q[17]), "=r"(q[18]), "=r"(q[19]), "=r"(q[20]), "=r"(q[21]), "=r"(q[22]), "=r"(q[23]),
                   "=r"(q[24]), "=r"(q[25]), "=r"(q[26]), "=r"(q[27]), "=r"(q[28]), "=r"(q[29]), "=r"(q[30]), "=r"(q[31])
                 : "r"(taddr));
}
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float (&v)[N]) {
    uint32_t r[N];
#pragma unroll
    for (int h = 0; h < N; h += 32) tmem_ld32_issue(taddr + h, r + h);
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
                 "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
                   "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]),
                   "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]),
                   "r"(v[30]), "r"(v[31])
                 : "memory");
}

// 8 codes as 8 float16 values c s + z, each rounded once: pairs (0, 4), (1, 5), (2, 6), (3, 7); s2 and z2 for the two of a pair.
__device__ __forceinline__ uint4 values_of(uint32_t w, uint32_t s2, uint32_t z2) {
    const __half2 s = *reinterpret_cast<__half2*>(&s2), z = *reinterpret_cast<__half2*>(&z2);
    const uint32_t k1024 = 0x64006400u, k16th = 0x2c002c00u, k64 = 0xd400d400u;       // 1024, 1/16, -64
    uint32_t out[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t u = i < 2 ? w : w >> 8;
        uint32_t bits = (u & (i & 1 ? 0x00f000f0u : 0x000f000fu)) | k1024;          // 1024 + c, or 1024 + 16 c
        const __half2 x = *reinterpret_cast<__half2*>(&bits);
        const __half2 c = i & 1 ? __hfma2(x, *reinterpret_cast<const __half2*>(&k16th), *reinterpret_cast<const __half2*>(&k64))
                                : __hsub2(x, *reinterpret_cast<const __half2*>(&k1024));
        const __half2 v = __hfma2(c, s, z);
        out[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
}

// (s, z) of one token's groups as they lie: N words
template <int N>
__device__ __forceinline__ void load_steps(const unsigned char* p, uint32_t (&v)[N]) {
    if constexpr (N == 1) v[0] = *reinterpret_cast<const uint32_t*>(p);
    else if constexpr (N == 2) { const uint2 x = *reinterpret_cast<const uint2*>(p); v[0] = x.x; v[1] = x.y; }
    else { const uint4 x = *reinterpret_cast<const uint4*>(p); v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; }
}

template <int D, int G>
struct Shape {
    static constexpr int NB = D / 64;
    static constexpr uint32_t Q_BYTES = 128 * D * 2, KV_BYTES = BN * D * 2;       // of 128 rows, of a tile of K or V
    static constexpr uint32_t Q = 0, KV = 2 * Q_BYTES, NAN_KEYS = KV + STAGES * 2 * KV_BYTES;
    static constexpr uint32_t CODES = NAN_KEYS + STAGES * 8 * 4 * 2;                                      // (NAN_KEYS: [stage][group][16 keys] 16 bits)
    static constexpr uint32_t BARS = CODES + MAKERS * RAW * i4_cache_tile_bytes(D, G);
    static constexpr uint32_t BYTES = BARS + 8 * (24 + 4 * STAGES + MAKERS * RAW);
    static constexpr uint32_t TMEM = 512;      // scores: 64 columns of tile j of half m at 128 m + 64 (j % 2); outputs from 256 on
};

template <int D, int G>
__global__ void __launch_bounds__(THREADS) int4_attention_tc_kernel(Args a) {
    using S = Shape<D, G>;
    constexpr int NB = S::NB, NG = D / G, GB = 64 / G, TILE = i4_cache_tile_bytes(D, G);
    extern __shared__ __align__(1024) unsigned char sm[];
    const uint32_t base = i4_smem(sm);
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + S::BARS);
    uint64_t &q_full = bars[0], *pv_done = bars + 1, *s_full = bars + 3, *p_full = bars + 7;        // s_full, p_full: [half][tile % 2]
    uint64_t *k_full = bars + 11, *k_empty = k_full + STAGES, *v_full = k_empty + STAGES, *v_empty = v_full + STAGES;
    uint64_t* raw_full = v_empty + STAGES;              // [maker][RAW]
    uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(raw_full + MAKERS * RAW);
    uint64_t* drained = raw_full + MAKERS * RAW + 1;    // [half]: all its products have ended
    unsigned short* nan_keys = reinterpret_cast<unsigned short*>(sm + S::NAN_KEYS);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    ce_pdl_wait();

    // rows row0 .. + rows of the (token, head) pairs of a tile of 64 tokens; later tiles, which see more keys, first
    const int kvh = blockIdx.x, i_tile = (int)(gridDim.y - 1 - blockIdx.y), row0 = blockIdx.z * a.block_rows;
    const int b = a.tiles[2 * i_tile], q0 = a.tiles[2 * i_tile + 1], each = a.nh / a.nkv;
    const int t0 = a.q_start[b] + q0, n = a.q_start[b + 1] - a.q_start[b], tokens = min(64, n - q0);
    const int rows = min(a.block_rows, tokens * each - row0), pos0 = a.ctx_len[b] - n + q0;
    if (rows <= 0) return;
    const int p_first = pos0 + row0 / each, p_last = pos0 + (row0 + rows - 1) / each;
    const int block_lo = a.window > 0 ? max(0, p_first - a.window + 1) : 0, k_begin = block_lo / BN * BN;
    const int n_kv = p_last < block_lo ? 0 : (p_last - k_begin) / BN + 1, mts = rows > 128 ? 2 : 1;
    const int* table = a.block_table + (size_t)a.seq_slot[b] * a.max_pages;
    const bool refused = (base & 1023u) != 0;           // cannot happen with dynamic shared memory alone; refuse rather than mis-swizzle
    if (refused && threadIdx.x == 0) atomicCAS(a.status, 0, 69);
    if (n_kv == 0 || refused) {
        for (int x = threadIdx.x; x < rows * (D / 8); x += THREADS) {
            const int rho = row0 + x / (D / 8), tok = rho / each;
            *reinterpret_cast<uint4*>(a.out + ((size_t)(t0 + tok) * a.nh + kvh * each + rho - tok * each) * D + x % (D / 8) * 8) = make_uint4(0, 0, 0, 0);
        }
        return;
    }
    if (threadIdx.x == 0) {
        mbar_init(&q_full, SOFTMAX);
        for (int s = 0; s < STAGES; ++s) { mbar_init(&k_full[s], 4); mbar_init(&k_empty[s], mts); mbar_init(&v_full[s], 4); mbar_init(&v_empty[s], mts); }
        for (int i = 0; i < MAKERS * RAW; ++i) mbar_init(&raw_full[i], 1);
        for (int i = 0; i < 4; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 4); }
        for (int i = 0; i < 2; ++i) { mbar_init(&pv_done[i], 1); mbar_init(&drained[i], 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(i4_smem(&tmem_slot)), "r"(S::TMEM));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    ce_pdl_launch_dependents();
    const uint32_t tmem = tmem_slot;

    if (warp < 2) {
        const int m = warp;
        if (m < mts) {
            // ---- the products of 128 rows: S(0) and S(1), then O += P(j) V(j) and S(j + 2), which takes the place of P(j)
            const uint32_t idesc_s = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | (8u << 24);
            const uint32_t idesc_pv = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | (8u << 24);
            const uint32_t tmem_s = tmem + m * 128, tmem_o = tmem + 256 + m * D, q_addr = base + S::Q + m * S::Q_BYTES;
            int where = 62;
            bool ok = i4_warp_wait(&q_full, 0);
            auto scores = [&](int j) {
                const int s = j % STAGES;
                where = 63;
                ok = i4_warp_wait(&k_full[s], (j / STAGES) & 1);
                if (!ok) return;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t k_addr = base + S::KV + s * 2 * S::KV_BYTES;
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                    umma(tmem_s + (j & 1) * BN, desc_kmajor(q_addr + (kk / 4) * 16384 + (kk % 4) * 32), desc_kmajor(k_addr + (kk / 4) * 8192 + (kk % 4) * 32),
                         idesc_s, kk > 0 ? 1u : 0u);
                umma_commit(&s_full[2 * m + (j & 1)]);
                umma_commit(&k_empty[s]);
            };
            if (ok) scores(0);
            if (ok && n_kv > 1) scores(1);
            for (int j = 0; j < n_kv && ok; ++j) {
                const int s = j % STAGES;
                where = 65;
                ok = i4_warp_wait(&v_full[s], (j / STAGES) & 1) && i4_warp_wait(&p_full[2 * m + (j & 1)], (j >> 1) & 1);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t v_addr = base + S::KV + s * 2 * S::KV_BYTES + S::KV_BYTES;
#pragma unroll
                for (int kk = 0; kk < BN / 16; ++kk)
                    umma_ts(tmem_o, tmem_s + (j & 1) * BN + kk * 8, desc_mnmajor(v_addr + kk * 16 * 128, 8192), idesc_pv, (j > 0 || kk > 0) ? 1u : 0u);
                umma_commit(&pv_done[m]);
                umma_commit(&v_empty[s]);
                if (j + 2 < n_kv) {
                    // (products of different shapes are not promised to run in order: P(j) has been read before its place is written again)
                    where = 64;
                    ok = i4_warp_wait(&pv_done[m], j & 1);
                    if (ok) scores(j + 2);
                }
            }
            if (!ok && lane == 0) atomicCAS(a.status, 0, where);
            // (whoever gave up: no product is under way when tensor and shared memory become another's)
            umma_commit(&drained[m]);
            i4_warp_wait(&drained[m], 0);
        }
        __syncwarp();
    } else if (warp < 2 + MAKERS) {
        // ---- the tiles of 16 keys, four to every 64, dealt out to the warps in turn: a tile's keys, then its values
        const int maker = warp - 2, r = lane >> 2, l = lane & 3, per_page = a.page_size >> 4, runs = 4 * n_kv;
        unsigned char* raw = sm + S::CODES + maker * RAW * TILE;
        uint64_t* raw_bars = raw_full + maker * RAW;
        auto run_of = [&](int i) { return maker + i * MAKERS; };
        auto first_key = [&](int run) { return k_begin + run * 16; };
        auto needed = [&](int run) { return run < runs && first_key(run) <= p_last && first_key(run) + 15 >= block_lo; };
        // where 32 of the warp's tiles lie, one a lane
        int looked = 0;
        const unsigned char* place = a.pages;
        auto look_up = [&](int from) {
            looked = from;
            const int run = run_of(from + lane), t = first_key(run) >> 4, pi = t / per_page;
            int page = !needed(run) ? 0 : pi < a.max_pages ? table[pi] : -1;
            if (page < 0 || page >= a.num_pages) { atomicExch(a.status, 4); page = 0; }      // (the step's results are not used)
            place = a.pages + (((size_t)page * a.nkv + kvh) * per_page + (t - pi * per_page)) * TILE;
        };
        auto fetch = [&](int i) {
            if (i >= looked + 32) look_up(i);
            const unsigned char* src = reinterpret_cast<const unsigned char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(place), i - looked));
            if (lane == 0 && needed(run_of(i))) i4_copy(raw + i % RAW * TILE, src, TILE, &raw_bars[i % RAW]);
        };
        look_up(0);
        for (int i = 0; i < RAW; ++i) fetch(i);
        I4Ring<RAW> ring;
        auto wait = [&](int at, uint32_t parity) { return i4_warp_wait(&raw_bars[at], parity); };
        bool ok = true;
        int next = 0;                                   // the tile whose copy is the next to be waited for
        for (int i = 0; run_of(i) < runs; ++i) {
            const int run = run_of(i), j = run >> 2, s = j % STAGES, key0 = first_key(run), part = run & 3;
            const bool here = needed(run), cut = !here || key0 < block_lo || key0 + 15 > p_last;
            const unsigned char* from = raw + i % RAW * TILE;
            unsigned char* to = sm + S::KV + s * 2 * S::KV_BYTES;
            uint4 kw[NB], vw[NB];
            uint32_t ks[2][NG], vs[4][NG];              // steps of tokens r and r + 8; of the four tokens of this lane's words of values
            auto token_of = [&](int e) { return 2 * l + (e & 1) + 8 * (e >> 1); };
            if (here) {
                ok = ring.landed(i, wait);
                if (!ok) break;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    kw[nb] = *reinterpret_cast<const uint4*>(from + nb * 512 + lane * 16);
                    vw[nb] = *reinterpret_cast<const uint4*>(from + 8 * D + nb * 512 + lane * 16);
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) load_steps<NG>(from + 16 * D + (r + 8 * e) * NG * 4, ks[e]);
#pragma unroll
                for (int e = 0; e < 4; ++e) load_steps<NG>(from + 16 * D + 64 * NG + token_of(e) * NG * 4, vs[e]);
            } else {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) kw[nb] = vw[nb] = make_uint4(0, 0, 0, 0);
            }
            __syncwarp();
            fetch(i + RAW);
            next = i + 1;
            if (cut) {                                  // the steps of what lies beyond the block's keys are zeros: anything may lie there
                auto in = [&](int token) { return here && key0 + token >= block_lo && key0 + token <= p_last; };
#pragma unroll
                for (int g = 0; g < NG; ++g) {
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        if (!in(r + 8 * e)) ks[e][g] = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!in(token_of(e))) vs[e][g] = 0;
                }
            }
            if (j >= STAGES) ok = i4_warp_wait(&k_empty[s], (j / STAGES - 1) & 1);
            if (!ok) break;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < 4; ++e) {           // words of tokens r and r + 8, first and second 32 channels
                    const int half = e >> 1, row = 16 * part + r + 8 * (e & 1);
                    const uint32_t word = e == 0 ? kw[nb].x : e == 1 ? kw[nb].y : e == 2 ? kw[nb].z : kw[nb].w;
                    const uint32_t p = ks[e & 1][(64 * nb + 32 * half) / G];
                    *reinterpret_cast<uint4*>(to + nb * 8192 + row * 128 + (((half * 4 + l) ^ (row & 7)) << 4)) =
                        values_of(word, __byte_perm(p, p, 0x1010), __byte_perm(p, p, 0x3232));
                }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&k_full[s]);
            if (j >= STAGES) ok = i4_warp_wait(&v_empty[s], (j / STAGES - 1) & 1);
            if (!ok) break;
            // groups of values that are not numbers: noted, and zeros in the tile
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                uint32_t bad = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (isnan(i4_unpack(vs[e][g]).x)) { bad |= 1u << token_of(e); vs[e][g] = 0; }
                if (__any_sync(0xffffffffu, bad)) {
                    bad |= __shfl_xor_sync(0xffffffffu, bad, 1);
                    bad |= __shfl_xor_sync(0xffffffffu, bad, 2);
                }
                if (lane == 0) nan_keys[(s * 8 + g) * 4 + part] = (unsigned short)bad;
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int row = 16 * part + token_of(e);
                    const uint32_t word = e == 0 ? vw[nb].x : e == 1 ? vw[nb].y : e == 2 ? vw[nb].z : vw[nb].w;
                    const uint32_t lo = vs[e][nb * GB], hi = vs[e][nb * GB + GB - 1];      // a word's halves lie 32 channels apart
                    *reinterpret_cast<uint4*>(to + S::KV_BYTES + nb * 8192 + row * 128 + ((r ^ (row & 7)) << 4)) =
                        values_of(word, __byte_perm(lo, hi, 0x5410), __byte_perm(lo, hi, 0x7632));
                }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&v_full[s]);
        }
        if (!ok) {
            if (lane == 0) atomicCAS(a.status, 0, 61);
            ring.drain(next, [&](int i) { return needed(run_of(i)); }, wait);
        }
    } else {
        // ---- softmax: a row a thread
        const int m = (warp - 2 - MAKERS) >> 2, quad = warp & 3, row = quad * 32 + lane, rr = m * 128 + row;
        const bool valid = rr < rows;
        const int rho = row0 + rr, tok = rho / each, pos = valid ? pos0 + tok : -1;
        const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
        const size_t head_row = valid ? (size_t)(kvh * each + rho - tok * each) : 0;
        float row_scale;
        {
            // the row, brought into [2^14, 2^15), its channels in the order of the keys'
            uint4 x[D / 8];
            const uint4* src = reinterpret_cast<const uint4*>(a.q + (size_t)(t0 + (valid ? tok : 0)) * a.q_stride + head_row * D);
            float largest = 0.f;
            bool finite = true;
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                x[c] = valid ? src[c] : make_uint4(0, 0, 0, 0);
                const uint32_t words[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float u = __uint_as_float(words[i] << 16), v = __uint_as_float(words[i] & 0xffff0000u);
                    largest = fmaxf(largest, fmaxf(fabsf(u), fabsf(v)));
                    finite = finite && fabsf(u) <= 3.402823466e38f && fabsf(v) <= 3.402823466e38f;
                }
            }
            const float up = i4_row_scale(finite ? largest : INFINITY);
            row_scale = i4_normal(a.scale_log2 / up);
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                const uint32_t words[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
                float f[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(words[i] << 16) * up; f[2 * i + 1] = __uint_as_float(words[i] & 0xffff0000u) * up; }
                *reinterpret_cast<uint4*>(sm + S::Q + m * S::Q_BYTES + (c >> 3) * 16384 + row * 128 + (((c & 7) ^ (row & 7)) << 4)) =
                    make_uint4(i4_pack(f[0], f[4]), i4_pack(f[1], f[5]), i4_pack(f[2], f[6]), i4_pack(f[3], f[7]));
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full);
        }
        if (m < mts) {
            const uint32_t lane_base = (uint32_t)(quad * 32) << 16, tmem_s = tmem + m * 128 + lane_base, tmem_o = tmem + 256 + m * D + lane_base;
            float m_run = -INFINITY, l_run = 0.f;
            uint32_t nan_groups = 0;
            bool ok = true;
            int where = 66;
            for (int j = 0; j < n_kv; ++j) {
                const int k0 = k_begin + j * BN;
                where = 66;
                if (!i4_warp_wait(&s_full[2 * m + (j & 1)], (j >> 1) & 1)) { ok = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                float sv[BN];
                tmem_ld<BN>(tmem_s + (j & 1) * BN, sv);
                const bool full = k0 >= lo && k0 + BN - 1 <= pos;
                if (!full) {
#pragma unroll
                    for (int i = 0; i < BN; ++i)
                        if (k0 + i < lo || k0 + i > pos) sv[i] = -INFINITY;
                }
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < BN; i += 4) {
                    mx4[0] = fmaxf(mx4[0], sv[i]); mx4[1] = fmaxf(mx4[1], sv[i + 1]);
                    mx4[2] = fmaxf(mx4[2], sv[i + 2]); mx4[3] = fmaxf(mx4[3], sv[i + 3]);
                }
                // the reference lies LIFT below the largest score it was set by, and is moved when a score passes that by HEADROOM
                const float m_tile = __fmaf_rd(fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])), row_scale, -LIFT);
                const bool raise = m_tile > m_run + HEADROOM || (m_run == -INFINITY && m_tile != -INFINITY);
                const float m_new = raise ? m_tile : m_run, m_use = m_new == -INFINITY ? 0.f : m_new;
                const float alpha = raise ? ce_exp2_fast(m_run - m_use) : 1.0f;
                float2 sum2 = make_float2(0.f, 0.f);
                uint32_t packed[BN / 2];
                const float2 scale2 = make_float2(row_scale, row_scale), minus_m = make_float2(-m_use, -m_use);
                auto weights = [&](auto cut) {
#pragma unroll
                    for (int i = 0; i < BN; i += 2) {
                        float2 t = __ffma2_rn(make_float2(sv[i], sv[i + 1]), scale2, minus_m);
                        if (cut()) t = make_float2(i4_min(t.x, LIFT + HEADROOM), i4_min(t.y, LIFT + HEADROOM));
                        const float2 p = make_float2(ce_exp2_fast(t.x), ce_exp2_fast(t.y));
                        sum2 = __fadd2_rn(sum2, p);
                        packed[i / 2] = i4_pack(p.x, p.y);
                    }
                };
                if (__all_sync(0xffffffffu, fabsf(m_use) < COARSE)) weights(std::false_type());
                else weights(std::true_type());
                l_run = l_run * alpha + (sum2.x + sum2.y);
                m_run = m_new;
                // the probabilities, where the scores were: two keys a column
                tmem_st32(tmem_s + (j & 1) * BN, packed);
                if (j > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
                    // (the product of tile j - 2 is done: this tile's scores were issued behind it)
                    where = 67;
                    if (!i4_warp_wait(&pv_done[m], (j - 1) & 1)) { ok = false; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        float o[32];
                        uint32_t back[32];
                        tmem_ld<32>(tmem_o + c, o);
#pragma unroll
                        for (int i = 0; i < 32; ++i) back[i] = __float_as_uint(o[i] * alpha);
                        tmem_st32(tmem_o + c, back);
                    }
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                // values that are no numbers among this tile's keys
                where = 68;
                const int s = j % STAGES;
                if (!i4_warp_wait(&v_full[s], (j / STAGES) & 1)) { ok = false; break; }
                const unsigned long long* bad = reinterpret_cast<const unsigned long long*>(nan_keys + s * 8 * 4);
                unsigned long long any = 0;
#pragma unroll
                for (int g = 0; g < NG; ++g) any |= bad[g];
                if (any) {
                    unsigned long long seen = ~0ull;
                    if (pos < k0) seen = 0;
                    else if (pos - k0 < 63) seen &= (2ull << (pos - k0)) - 1;
                    if (lo > k0) seen &= lo - k0 > 63 ? 0ull : ~0ull << (lo - k0);
#pragma unroll
                    for (int g = 0; g < NG; ++g)
                        if (bad[g] & seen) nan_groups |= 1u << g;
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[2 * m + (j & 1)]);
            }
            if (ok) {
                where = 67;
                // the last two products may both be under way, and a parity tells one from the next only
                ok = (n_kv < 2 || i4_warp_wait(&pv_done[m], (n_kv - 2) & 1)) && i4_warp_wait(&pv_done[m], (n_kv - 1) & 1);
            }
            if (!ok) {
                if (lane == 0) atomicCAS(a.status, 0, where);
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (ok) {
                const float inv = l_run == 0.f ? 0.f : 1.0f / l_run;
                __nv_bfloat16* dst = a.out + ((size_t)(t0 + tok) * a.nh + head_row) * D;
#pragma unroll 1
                for (int nb = 0; nb < NB; ++nb) {
                    float o[64];
                    tmem_ld<64>(tmem_o + nb * 64, o);
                    if (valid) {
#pragma unroll
                        for (int c = 0; c < 64; c += 8) {
                            const bool nan = nan_groups >> ((64 * nb + c) / G) & 1;
                            uint32_t v[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                // channel 32 e + 4 r + n of a block lies at 8 r + 2 n + e
                                const int c0 = c + 2 * i, c1 = c0 + 1;
                                const float x = o[(c0 & 31) / 4 * 8 + (c0 & 3) * 2 + (c0 >> 5)] * inv, y = o[(c1 & 31) / 4 * 8 + (c1 & 3) * 2 + (c1 >> 5)] * inv;
                                __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
                                v[i] = nan ? 0x7fff7fffu : *reinterpret_cast<uint32_t*>(&h);
                            }
                            *reinterpret_cast<uint4*>(dst + nb * 64 + c) = make_uint4(v[0], v[1], v[2], v[3]);
                        }
                    }
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        }
    }
    __syncthreads();
    if (warp == 0) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::TMEM));
    }
}

template <int D, int G>
int run(const Args& a, dim3 grid, cudaStream_t stream) {
    static std::atomic<unsigned long long> done{0};
    cudaError_t e = ce_allow_smem(done, int4_attention_tc_kernel<D, G>, Shape<D, G>::BYTES);
    if (e == cudaSuccess) {
        ce_note("int4_attention_tc_kernel");
        e = ce_launch(int4_attention_tc_kernel<D, G>, grid, dim3(THREADS), Shape<D, G>::BYTES, stream, a);
    }
    if (e != cudaSuccess) { (void)cudaGetLastError(); return ce_fail(CE_ERR_CUDA, "int4_attention_tc: %s", cudaGetErrorString(e)); }
    return ce_check_launch("int4_attention_tc");
}

}  // namespace

// Rows of a block: a tile's 64 tokens by ``each`` heads in equal shares of at most 256
static int tc_rows(int each) {
    const int subs = (64 * each + 255) / 256;
    return (64 * each + subs - 1) / subs;
}
// Blocks that a KV head of a tile of 64 tokens takes; 0: not sizes of this kernel (operands that start between 16-byte boundaries are not either)
extern "C" int ce_int4_attention_tc_blocks(int each, int d) { return d == 64 || d == 128 ? (64 * each + tc_rows(each) - 1) / tc_rows(each) : 0; }

// q, q_stride, pages, out, seq_slot, q_start, ctx_len, block_table, status, tiles, n_tiles, nh, nkv, d, group, page_size, max_pages, num_pages,
// window, scale, stream.  The checks of ce_int4_attention come first: it calls this.
int ce_int4_attention_tc(const void* q, long long q_stride, const void* pages, void* out, const int* seq_slot, const int* q_start, const int* ctx_len,
                         const int* block_table, int* status, const int* tiles, int n_tiles, int nh, int nkv, int d, int group, int page_size,
                         int max_pages, int num_pages, int window, float scale, cudaStream_t stream) {
    const int each = nh / nkv, blocks = ce_int4_attention_tc_blocks(each, d);
    if (!blocks || n_tiles > 65535 || blocks > 65535 || (((uintptr_t)q | (uintptr_t)out) & 15) || q_stride % 8)
        return ce_fail(CE_ERR_SIZE, "int4_attention_tc: not sizes of this kernel");
    Args a{(const __nv_bfloat16*)q, (__nv_bfloat16*)out, (const unsigned char*)pages, seq_slot, q_start, ctx_len, block_table, tiles, status,
           q_stride, nh, nkv, page_size, max_pages, num_pages, window, tc_rows(each), scale * 1.4426950408889634f};
    const dim3 grid(nkv, n_tiles, blocks);
    if (d == 64) return group == 32 ? run<64, 32>(a, grid, stream) : run<64, 64>(a, grid, stream);
    return group == 32 ? run<128, 32>(a, grid, stream) : run<128, 64>(a, grid, stream);
}
