// Attention of a step of single tokens whose rows are the beams of requests: the beams of a request share the keys of their prompt and have
// some of their own.  bf16, paged, grouped-query, compiled for one RI_HEAD_DIM (a multiple of 16, at most 256).
//
//     out[r, h] = sum_k softmax_k(scale q[r, h] . K[k]) V[k],   k over [kv_len[r] - window, kv_len[r])
//
// Keys before shared_len[g] are the same for every row of group g, whose rows follow one another: one CTA reads a range of them, by the
// first row's table, for all beams x heads of a key head, which are the M dimension of the matrix products.  Keys from there on are read
// by each row's own table, by a warp for one key head's heads.  Both leave partial results (a sum weighted by 2^(score - maximum), its
// log-sum-exp in base 2) that a second kernel joins.  RustInfer's decode attention reads a request's keys for that request alone
// (crates/infer-backend-cuda/src/kernels/flash_attn_gqa/flash_attn_paged_decode.cu:75-340).
//
// What bounds it is the cache's stream: shared keys and values once a request, the beams' own once a beam.  Scores, maxima, sums and
// outputs are 32-bit.  A weight enters the product with the values as two bf16 pieces that add up to it to 2^-17 of itself: rounded to one
// piece it would be off by up to 2^-9, as much as the stored output's own rounding.
//
// Shared keys come by TMA where the head size is 64 or 128 and a page holds 8, 16, 32 or a multiple of 64 keys (a box a page and 64 columns,
// each from a lane of its own; the 128-byte swizzle, which ldmatrix reads through), else by cp.async: half of the loop's instructions were
// the latter's addresses.
#include "common.cuh"
#include <cuda.h>
#include <mutex>

#ifndef RI_HEAD_DIM
#error "compile with -DRI_HEAD_DIM=<head size>"
#endif

namespace {
constexpr int HD = RI_HEAD_DIM;
static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "beam attention: head size multiple of 16, at most 256");
constexpr int ROW = HD + 8;                                // padded rows: 16 bytes on, ldmatrix meets no bank twice
constexpr int OROW = HD + 8;                               // rows of outputs in shared memory: pairs of lanes apart
constexpr int CH = HD / 8;                                 // 16-byte pieces a row
constexpr int KS = HD / 16;
constexpr int NT = HD / 8;
constexpr int WARPS = 4;
constexpr int THREADS = 32 * WARPS;
constexpr int CTAS = HD <= 64 ? 4 : HD <= 128 ? 2 : 1;     // CTAs an SM that registers and shared memory are cut for
constexpr int MAX_BEAMS = 64;
constexpr int OWN_KEYS = 16;                               // keys of its own a row's warp takes at a time
constexpr int OWN_STAGES = 2;                              // of which so many are on their way
constexpr bool BY_TMA = HD == 64 || HD == 128;
constexpr int TKB_OR_1 = BY_TMA ? HD / 64 : 1;             // 64-column blocks of a head
constexpr unsigned SPIN_LIMIT = 1u << 20;
// A weight is 2^(fma(score, scale, -maximum)), which leaves out the rounding that the maximum, a product itself, has had.  That is a factor of a
// tile's weights, and next to nothing, until it passes the exponents' range: beyond FAR the scores are rounded first, and the largest weight is 1.
constexpr float FAR = 16777216.f;

constexpr int KT = 64;                                     // keys of a tile
constexpr int STAGES = 2;
// (us.  8 x 8 beams, heads of 64, behind 4,096 / 16,384 keys, before a range's start and end took 3 us less: 4 warps, 4 CTAs an SM 28 / 69; 8 warps,
// 2 CTAs, tiles of 128, 3 stages 28 / 79; 4 warps and 3 CTAs 32 / 83, 5 CTAs 31 / 76.  4 x 16 beams, heads of 128, behind up to 9,001 / 36,004:
// 4 warps, 2 CTAs 52 / 141; 8 warps, 2 CTAs 59 / 145)
// rows of shared keys are split over RTILES warps, a tile's keys over the others
template <int RTILES> constexpr int key_groups() { return WARPS / RTILES < KT / 16 ? WARPS / RTILES : KT / 16; }

__device__ __forceinline__ void cp_async16(void* smem, const void* gmem, bool valid) {
    const unsigned s = (unsigned)__cvta_generic_to_shared(smem);
    const int n = valid ? 16 : 0;                          // 0 bytes read: the 16 bytes are filled with zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(s), "l"(gmem), "r"(n));
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N)); }
// by 32-bit shared addresses: through pointers every fragment cost half a dozen instructions of address
__device__ __forceinline__ void ldmatrix_x4(unsigned (&r)[4], unsigned s) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s));
}
__device__ __forceinline__ void ldmatrix_x4_trans(unsigned (&r)[4], unsigned s) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {            // 2 ulp
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint64_t* bar) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t* bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
// bounded: false after SPIN_LIMIT tries
__device__ __forceinline__ bool bar_wait(uint64_t* bar, unsigned parity) {
#pragma unroll 1
    for (unsigned i = 0; i < SPIN_LIMIT; ++i) {
        unsigned ok;
        asm volatile("{\n\t.reg .pred p;\n\t"
                     "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                     "selp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
        if (ok) return true;
        if (i > 1024) __nanosleep(64);
    }
    return false;
}
__device__ __forceinline__ void tma_load_2d(void* smem, const CUtensorMap* map, uint64_t* bar, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(smem_u32(smem)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y) : "memory");
}
// d (8 rows x 8 columns of a 16 x 8 product whose lower rows are zero) += a b
__device__ __forceinline__ void mma_8rows(float (&d)[2], unsigned a0, unsigned a2, unsigned b0, unsigned b1) {
    [[maybe_unused]] float x, y;
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%5}, {%7,%8}, {%0,%1,%9,%9};\n"
                 : "+f"(d[0]), "+f"(d[1]), "=f"(x), "=f"(y)
                 : "r"(a0), "r"(0u), "r"(a2), "r"(b0), "r"(b1), "f"(0.f));
}
// two weights as bf16 pairs: the rounded weights, and what the rounding left
__device__ __forceinline__ void two_pieces(float a, float b, unsigned& high, unsigned& low) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    const __nv_bfloat162 l = __floats2bfloat162_rn(a - __low2float(h), b - __high2float(h));
    high = *reinterpret_cast<const unsigned*>(&h);
    low = *reinterpret_cast<const unsigned*>(&l);
}

struct Args {
    const bf16* q;
    int q_stride;
    const bf16* cache;
    const int* table;
    int table_stride, table_keys;                         // keys a row of the table has pages for
    int pages;                                             // of the cache: a number outside stands for a page of zeros
    const int* kv_len;
    const int* shared_len;
    int beams, Hq, Hkv, page_size;
    float scale_log2;
    int window, groups, shared_splits, own_splits, target;
    float* part_o;
    float* part_lse;
    int* error;
    int box_rows;                                          // rows of a TMA box: a page's, or a tile's of a large one
};

// A row's keys: no more than its table has pages for, whatever it is said to have
__device__ __forceinline__ int keys_of(const Args& a, int r) { return min(max(0, a.kv_len[r]), a.table_keys); }

// The keys the rows of group g share, as [from, to): what its table gives up to shared_len, if every row sees all of them; else none (the
// rows then read all their keys by their own tables).  Every thread of a warp gets it.
__device__ __forceinline__ void shared_range(const Args& a, int g, int& from, int& to) {
    const int lane = threadIdx.x & 31;
    const int s = max(0, a.shared_len[g]);
    const int first = keys_of(a, g * a.beams);
    const int lo = a.window > 0 ? max(0, first - a.window) : 0;
    bool same = true;
    for (int b = lane; b < a.beams; b += 32) {
        const int n = keys_of(a, g * a.beams + b);
        same = same && n >= s && (a.window <= 0 || max(0, n - a.window) == lo);
    }
    same = __all_sync(0xffffffffu, same);
    from = lo;
    to = same && s > lo ? s : lo;
}

// Keys [lo, hi) by table row `bt` for the rows m0 .. m0 + m_count - 1 (of beams x heads) of group g, RTILES tiles of 16 rows in one CTA.  Tiles
// lie where the multiples of their size do, so that a page's keys lie in one.
template <int RTILES, bool TMA>
__device__ __forceinline__ void attend(const Args& a, const CUtensorMap* map, unsigned char* smem, int g, int kvh, int m0, int m_count, const int* bt,
                                       int lo, int hi, int part) {
    constexpr int KG = key_groups<RTILES>();
    static_assert(RTILES * KG == WARPS, "a warp without a part would read queries that are not there");
    constexpr int WK = KT / KG;                            // keys a warp takes of a tile
    constexpr int NK = WK / 8;
    constexpr int PIECES = (KT * CH + THREADS - 1) / THREADS;      // 16-byte pieces of a tile's keys a thread fetches
    constexpr int KROW = TMA ? HD : ROW;
    constexpr int STAGE = 2 * KT * KROW;                   // elements
    constexpr int KROW_BYTES = TMA ? 128 : ROW * 2;        // by TMA: of a block of 64 columns
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = a.Hq / a.Hkv, splits = a.shared_splits + a.own_splits;
    bf16* KVs = reinterpret_cast<bf16*>(smem);             // [STAGES][K | V][KT][KROW]
    bf16* Qs = KVs + STAGES * STAGE;                       // [RTILES * 16][ROW]
    uint64_t* full = reinterpret_cast<uint64_t*>(Qs + RTILES * 16 * ROW);
    const int rt = warp / KG, kg = warp % KG;
    // where a lane's fragments lie in a stage, in bytes: a row of keys and one of values.  By TMA, columns 16 ks on are an exclusive or away
    // (the swizzle's bits are the only ones below a row), 64 columns a block; else 32 bytes a step
    const int k_row = kg * WK + (lane & 7) + (lane >> 4) * 8, v_row = kg * WK + (lane & 15);
    const unsigned base = smem_u32(KVs), q_at = smem_u32(Qs) + ((rt * 16 + (lane & 15)) * ROW + (lane >> 4) * 8) * 2;
    const unsigned k_at = k_row * KROW_BYTES + (TMA ? ((((lane >> 3) & 1) ^ (k_row & 7)) << 4) : ((lane >> 3) & 1) * 16);
    const unsigned v_at = KT * KROW * 2 + v_row * KROW_BYTES + (TMA ? (((lane >> 4) ^ (v_row & 7)) << 4) : (lane >> 4) * 16);
    auto step = [&](unsigned at, int ks) -> unsigned {     // 16 columns a step
        if constexpr (TMA) return (at ^ ((ks & 3) << 5)) + (ks >> 2) * (KT * 128);
        else return at + ks * 32;
    };

    const int t0 = lo / KT, tiles = (hi + KT - 1) / KT - t0;
    const size_t head_step = (size_t)a.page_size * HD, value_step = (size_t)a.Hkv * head_step;
    const int shift = (a.page_size & (a.page_size - 1)) == 0 ? __ffs(a.page_size) - 1 : -1;
    // cp.async: where a thread's pieces of a tile lie, looked up a tile ahead of the fetch
    const bf16* from[PIECES];
    auto look_up = [&](int t) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int c = tid + i * THREADS, kk = c / CH, ch = c - kk * CH, key = (t0 + t) * KT + kk;
            from[i] = nullptr;
            if (c < KT * CH && key >= lo && key < hi) {
                const int blk = shift >= 0 ? key >> shift : key / a.page_size, page = bt[blk];
                if ((unsigned)page < (unsigned)a.pages)
                    from[i] = a.cache + ((size_t)page * 2 * a.Hkv + kvh) * head_step + (size_t)(key - blk * a.page_size) * HD + ch * 8;
            }
        }
    };
    // TMA, the first warp: a lane's box is keys or values, a page of the tile, 64 columns, the same in every tile; its page's number is read a
    // tile ahead.  No division in the loop: all other warps wait for this one (8 x 8 beams behind 4,000 keys 27.1 us with four a box, 25.6)
    const int boxes = KT / a.box_rows;                     // of keys, of 64 columns: no more than 8, and 32 in all
    const int box_kv = lane / (boxes * TKB_OR_1), box_rest = lane - box_kv * boxes * TKB_OR_1, box_c = box_rest / TKB_OR_1, box_kb = box_rest - box_c * TKB_OR_1;
    const bool small_pages = a.page_size < KT;             // a page a box; else a tile lies in one page
    const int box_row = (box_kv * a.Hkv + kvh) * a.page_size, page_rows = 2 * a.Hkv * a.page_size;
    const unsigned box_at = ((box_kv * TKB_OR_1 + box_kb) * KT + box_c * a.box_rows) * 128;
    int next_page = 0, next_off = 0;                       // of the tile that was looked up (nothing waits for the load before the fetch does)
    bool next_box = false;
    int blk = small_pages ? t0 * boxes : t0 * KT / a.page_size, off = small_pages ? 0 : t0 * KT % a.page_size;
    auto look_up_box = [&](int t) {                        // tiles in order
        const int key = (t0 + t) * KT + box_c * a.box_rows;
        next_box = box_kv < 2 && key < hi && key + a.box_rows > lo;        // boxes without a key in [lo, hi) are not fetched
        next_off = off;
        if (next_box) next_page = bt[blk + (small_pages ? box_c : 0)];
        if (small_pages) blk += boxes;
        else if ((off += KT) >= a.page_size) { off = 0; ++blk; }
    };
    auto fetch = [&](int t, int stage) {                   // tile t, which was looked up; looks up the next
        if constexpr (TMA) {
            if (warp == 0) {
                const int page = (unsigned)next_page > (unsigned)a.pages ? a.pages : next_page;      // outside the cache: rows behind the matrix, zeros
                const bool mine = next_box;
                const unsigned all = __ballot_sync(0xffffffffu, mine);
                if (lane == 0) bar_expect(&full[stage], (unsigned)__popc(all) * a.box_rows * 128);
                __syncwarp();
                if (mine)
                    tma_load_2d(reinterpret_cast<unsigned char*>(KVs + stage * STAGE) + box_at, map, &full[stage], box_kb * 64,
                                page * page_rows + box_row + next_off);
                if (t + 1 < tiles) look_up_box(t + 1);
            }
        } else {
            bf16* Ks = KVs + stage * STAGE;
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int c = tid + i * THREADS, kk = c / CH, ch = c - kk * CH;
                if (c < KT * CH) {
                    const bool ok = from[i] != nullptr;
                    const bf16* k = ok ? from[i] : a.cache;
                    cp_async16(Ks + kk * ROW + ch * 8, k, ok);
                    cp_async16(Ks + (KT + kk) * ROW + ch * 8, ok ? k + value_step : k, ok);
                }
            }
            if (t + 1 < tiles) look_up(t + 1);
        }
    };
    // queries, all on their way at once (loaded and stored one after the other they were half of the time to the first tile); the first
    // tile's group takes them in, by TMA they are their own
    for (int c = tid; c < RTILES * 16 * CH; c += THREADS) {
        const int r = c / CH, ch = c - r * CH, m = m0 + min(r, m_count - 1), b = m / G;
        cp_async16(Qs + r * ROW + ch * 8, a.q + (size_t)(g * a.beams + b) * a.q_stride + (size_t)(kvh * G + m - b * G) * HD + ch * 8, r < m_count);
    }
    if constexpr (TMA) cp_async_commit();
    if constexpr (TMA) {
        if (tid == 0) {
            for (int s = 0; s < STAGES; ++s) bar_init(&full[s]);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        if (warp == 0) {
            look_up_box(0);
            __syncwarp();
        }
    } else {
        look_up(0);
    }
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
        if (s < tiles) fetch(s, s);
        if constexpr (!TMA) cp_async_commit();
    }
    float o[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    if constexpr (TMA) cp_async_wait<0>();
    __syncthreads();                                       // queries are there, and the barriers

    unsigned parity = 0;
    for (int t = 0, stage = 0; t < tiles; ++t) {
        // the tile has come, and the one before it is used up
        if constexpr (TMA) {
            if (!__syncthreads_and(bar_wait(&full[stage], parity))) {
                // a wait ran out: the copies behind are waited for too, with the same limit, and the host is told
                for (int u = t; u < min(tiles, t + STAGES - 1); ++u) {
                    bar_wait(&full[stage], parity);
                    if (++stage == STAGES) { stage = 0; parity ^= 1u; }
                }
                if (tid == 0) atomicExch(a.error, 22);
                break;
            }
        } else {
            cp_async_wait<STAGES - 2>();
            __syncthreads();
        }
        if (t + STAGES - 1 < tiles) fetch(t + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
        if constexpr (!TMA) cp_async_commit();
        bf16* Vs = KVs + stage * STAGE + KT * KROW;
        const unsigned stage_at = base + stage * (STAGE * 2);
        if (++stage == STAGES) { stage = 0; parity ^= 1u; }
        const int kw0 = kg * WK, key0 = (t0 + t) * KT + kw0;
        if (key0 >= hi || key0 + WK <= lo) continue;
        const bool edge = key0 < lo || key0 + WK > hi;
        if constexpr (TMA) {
            if (edge) {
                // values of keys outside meet a weight of zero, but what lies there may be no number
                for (int i = lane; i < WK * CH; i += 32) {
                    const int r = i / CH, key = key0 + r;
                    const int col = (i - r * CH) * 8, row = kw0 + r;
                    if (key < lo || key >= hi)
                        *reinterpret_cast<uint4*>(Vs + (col >> 6) * (KT * 64) + row * 64 + ((((col & 63) >> 3) ^ (row & 7)) << 3)) = make_uint4(0u, 0u, 0u, 0u);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");     // ahead of the copy that the stage is used for next
                __syncwarp();
            }
        }
        float s[NK][4];
#pragma unroll
        for (int n = 0; n < NK; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            unsigned qf[4];                                // (from shared memory every tile: its registers make room for a second CTA)
            ldmatrix_x4(qf, q_at + ks * 32);
#pragma unroll
            for (int n2 = 0; n2 < NK / 2; ++n2) {
                unsigned kf[4];
                ldmatrix_x4(kf, step(stage_at + k_at, ks) + n2 * 16 * KROW_BYTES);
                mma_bf16(s[2 * n2], qf, kf[0], kf[1]);
                mma_bf16(s[2 * n2 + 1], qf, kf[2], kf[3]);
            }
        }
        float mx[2] = {-INFINITY, -INFINITY};
        if (edge) {
#pragma unroll
            for (int n = 0; n < NK; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = key0 + n * 8 + (lane & 3) * 2 + (e & 1);
                    if (key < lo || key >= hi) s[n][e] = -INFINITY;
                }
        }
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
        float alpha[2], muse[2], by[2] = {a.scale_log2, a.scale_log2};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2)) * a.scale_log2;
            const float mnew = fmaxf(m[i], mx[i]);
            muse[i] = mnew == -INFINITY ? 0.f : mnew;
            alpha[i] = ex2(m[i] - muse[i]);
            m[i] = mnew;
            l[i] *= alpha[i];
            if (fabsf(muse[i]) > FAR) {                    // rounded ahead of the subtraction
#pragma unroll
                for (int n = 0; n < NK; ++n) {
                    s[n][2 * i] = __fmul_rn(s[n][2 * i], a.scale_log2);
                    s[n][2 * i + 1] = __fmul_rn(s[n][2 * i + 1], a.scale_log2);
                }
                by[i] = 1.f;
            }
        }
        if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                o[n][0] *= alpha[0]; o[n][1] *= alpha[0];
                o[n][2] *= alpha[1]; o[n][3] *= alpha[1];
            }
        }
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[n][e] = ex2(fmaf(s[n][e], by[e >> 1], -muse[e >> 1]));
                l[e >> 1] += s[n][e];
            }
#pragma unroll
        for (int n2 = 0; n2 < NK / 2; ++n2) {
            unsigned ph[4], pl[4];
            two_pieces(s[2 * n2][0], s[2 * n2][1], ph[0], pl[0]);
            two_pieces(s[2 * n2][2], s[2 * n2][3], ph[1], pl[1]);
            two_pieces(s[2 * n2 + 1][0], s[2 * n2 + 1][1], ph[2], pl[2]);
            two_pieces(s[2 * n2 + 1][2], s[2 * n2 + 1][3], ph[3], pl[3]);
#pragma unroll
            for (int np = 0; np < NT / 2; ++np) {
                unsigned vf[4];
                ldmatrix_x4_trans(vf, step(stage_at + v_at, np) + n2 * 16 * KROW_BYTES);
                mma_bf16(o[2 * np], ph, vf[0], vf[1]);
                mma_bf16(o[2 * np + 1], ph, vf[2], vf[3]);
                mma_bf16(o[2 * np], pl, vf[0], vf[1]);
                mma_bf16(o[2 * np + 1], pl, vf[2], vf[3]);
            }
        }
    }
    if constexpr (!TMA) cp_async_wait<0>();

#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    auto part_of = [&](int r) -> size_t {                  // of row m0 + r
        const int mm = m0 + r, b = mm / G;
        return ((size_t)(g * a.beams + b) * a.Hq + kvh * G + mm - b * G) * splits + part;
    };
    if constexpr (KG == 1) {                               // a row's keys are one warp's: from its registers
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = rt * 16 + (lane >> 2) + 8 * i;
            if (r < m_count) {
                const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
                const size_t p = part_of(r);
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    *reinterpret_cast<float2*>(a.part_o + p * HD + n * 8 + (lane & 3) * 2) = make_float2(o[n][2 * i] * inv, o[n][2 * i + 1] * inv);
                if ((lane & 3) == 0) a.part_lse[p] = l[i] == 0.f ? -INFINITY : (m[i] == -INFINITY ? 0.f : m[i]) + log2f(l[i]);
            }
        }
    } else {
        // the warps' states through shared memory (the tiles are used up)
        __syncthreads();
        float* Os = reinterpret_cast<float*>(KVs);         // [WARPS][16][OROW]
        float* Ms = Os + WARPS * 16 * OROW;                // [WARPS][16]
        float* Ls = Ms + WARPS * 16;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = (lane >> 2) + 8 * i;
            float* orow = Os + (warp * 16 + r) * OROW + (lane & 3) * 2;
#pragma unroll
            for (int n = 0; n < NT; ++n) *reinterpret_cast<float2*>(orow + n * 8) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
            if ((lane & 3) == 0) { Ms[warp * 16 + r] = m[i]; Ls[warp * 16 + r] = l[i]; }
        }
        __syncthreads();
        constexpr int FOURS = RTILES * 16 * (HD / 4);      // four outputs a thread at a time
#pragma unroll
        for (int c0 = 0; c0 < FOURS; c0 += THREADS) {
            const int c = c0 + tid, r = c / (HD / 4), d = (c - r * (HD / 4)) * 4;
            if (c >= FOURS || r >= m_count) continue;
            const int w0 = (r >> 4) * KG, rr = r & 15;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < KG; ++w) M = fmaxf(M, Ms[(w0 + w) * 16 + rr]);
            const float muse = M == -INFINITY ? 0.f : M;
            float L = 0.f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < KG; ++w) {
                const float lw = Ls[(w0 + w) * 16 + rr], f = lw == 0.f ? 0.f : ex2(Ms[(w0 + w) * 16 + rr] - muse);
                L += lw * f;
                const float4 x = *reinterpret_cast<const float4*>(Os + ((w0 + w) * 16 + rr) * OROW + d);
                if (f != 0.f) { v.x += x.x * f; v.y += x.y * f; v.z += x.z * f; v.w += x.w * f; }
            }
            const float inv = L == 0.f ? 0.f : 1.f / L;
            const size_t p = part_of(r);
            *reinterpret_cast<float4*>(a.part_o + p * HD + d) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
            if (d == 0) a.part_lse[p] = L == 0.f ? -INFINITY : muse + log2f(L);                   // what is no number stays none
        }
    }
}

// A row's own keys [lo, hi) for up to 8 heads of one key head, by one warp: 16 keys at a time, the next keys on their way while the values are
// used and the other way round.
__device__ __forceinline__ void attend_own(const Args& a, unsigned char* smem, int r, int kvh, int head0, int heads, int lo, int hi, int part) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int splits = a.shared_splits + a.own_splits;
    constexpr int BUFFER = 2 * OWN_KEYS * ROW;             // elements: keys, then values
    bf16* Ks = reinterpret_cast<bf16*>(smem) + warp * OWN_STAGES * BUFFER;
    bf16* Vs = Ks + OWN_KEYS * ROW;
    const unsigned k_at = smem_u32(Ks) + (((lane & 7) + (lane >> 4) * 8) * ROW + ((lane >> 3) & 1) * 8) * 2;
    const unsigned v_at = smem_u32(Vs) + ((lane & 15) * ROW + (lane >> 4) * 8) * 2;
    const int* bt = a.table + (size_t)r * a.table_stride;
    const size_t head_step = (size_t)a.page_size * HD, value_step = (size_t)a.Hkv * head_step;
    // a lane's half of a row, 16 rows, two lanes each; its page's number is read a step ahead
    auto look_up = [&](int k0) -> int {
        const int key = k0 + (lane >> 1);
        return key < hi ? bt[key / a.page_size] : -1;
    };
    auto fetch = [&](bf16* to, int k0, int page, size_t step) {
        const int kk = lane >> 1;
        const bool there = k0 + kk < hi && (unsigned)page < (unsigned)a.pages;
        const bf16* src = there ? a.cache + ((size_t)page * 2 * a.Hkv + kvh) * head_step + (size_t)((k0 + kk) % a.page_size) * HD + step : a.cache;
#pragma unroll
        for (int ch = 0; ch < CH / 2; ++ch) {
            const int c = 2 * ch + (lane & 1);
            cp_async16(to + kk * ROW + c * 8, there ? src + c * 8 : src, there);
        }
        cp_async_commit();
    };
    const size_t p0 = ((size_t)r * a.Hq + head0) * splits + part;       // of the first head; the next is `splits` on
    if (lo >= hi) {
        if (lane < heads) a.part_lse[p0 + (size_t)lane * splits] = -INFINITY;
        return;
    }
    int page = look_up(lo), page_then = look_up(lo + OWN_KEYS), page_later = look_up(lo + 2 * OWN_KEYS);
    fetch(Ks, lo, page, 0);
    fetch(Vs, lo, page, value_step);
    fetch(Ks + BUFFER, lo + OWN_KEYS, page_then, 0);       // (keys from hi on: zeros, nothing is read)
    fetch(Vs + BUFFER, lo + OWN_KEYS, page_then, value_step);
    page = page_later;
    unsigned qf[KS][2];                                    // rows 0 to 7 alone
    {
        const int h = lane >> 2;
        const bf16* q = a.q + (size_t)r * a.q_stride + (size_t)(head0 + h) * HD + (lane & 3) * 2;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            qf[ks][0] = h < heads ? *reinterpret_cast<const unsigned*>(q + ks * 16) : 0u;
            qf[ks][1] = h < heads ? *reinterpret_cast<const unsigned*>(q + ks * 16 + 8) : 0u;
        }
    }
    float o[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = 0.f;
    float m = -INFINITY, l = 0.f;
    for (int k0 = lo, buffer = 0; k0 < hi; k0 += OWN_KEYS, buffer ^= BUFFER) {
        cp_async_wait<2 * OWN_STAGES - 1>();
        __syncwarp();
        float s[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            unsigned kf[4];
            ldmatrix_x4(kf, k_at + buffer * 2 + ks * 32);
            mma_8rows(s[0], qf[ks][0], qf[ks][1], kf[0], kf[1]);
            mma_8rows(s[1], qf[ks][0], qf[ks][1], kf[2], kf[3]);
        }
        __syncwarp();
        page_later = look_up(k0 + (OWN_STAGES + 1) * OWN_KEYS);
        if (k0 + OWN_STAGES * OWN_KEYS < hi) fetch(Ks + buffer, k0 + OWN_STAGES * OWN_KEYS, page, 0);
        else cp_async_commit();
        float mx = -INFINITY;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (k0 + n * 8 + (lane & 3) * 2 + e >= hi) s[n][e] = -INFINITY;
                mx = fmaxf(mx, s[n][e]);
            }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)) * a.scale_log2;
        const float mnew = fmaxf(m, mx), muse = mnew == -INFINITY ? 0.f : mnew, alpha = ex2(m - muse);
        m = mnew;
        l *= alpha;
#pragma unroll
        for (int n = 0; n < NT; ++n) { o[n][0] *= alpha; o[n][1] *= alpha; }
        const bool far = fabsf(muse) > FAR;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                s[n][e] = ex2(far ? __fmul_rn(s[n][e], a.scale_log2) - muse : fmaf(s[n][e], a.scale_log2, -muse));
                l += s[n][e];
            }
        unsigned ph[2], pl[2];
        two_pieces(s[0][0], s[0][1], ph[0], pl[0]);
        two_pieces(s[1][0], s[1][1], ph[1], pl[1]);
        cp_async_wait<2 * OWN_STAGES - 1>();
        __syncwarp();
#pragma unroll
        for (int np = 0; np < NT / 2; ++np) {
            unsigned vf[4];
            ldmatrix_x4_trans(vf, v_at + buffer * 2 + np * 32);
            mma_8rows(o[2 * np], ph[0], ph[1], vf[0], vf[1]);
            mma_8rows(o[2 * np + 1], ph[0], ph[1], vf[2], vf[3]);
            mma_8rows(o[2 * np], pl[0], pl[1], vf[0], vf[1]);
            mma_8rows(o[2 * np + 1], pl[0], pl[1], vf[2], vf[3]);
        }
        __syncwarp();
        if (k0 + OWN_STAGES * OWN_KEYS < hi) fetch(Vs + buffer, k0 + OWN_STAGES * OWN_KEYS, page, value_step);
        else cp_async_commit();
        page = page_later;
    }
    cp_async_wait<0>();
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    const int h = lane >> 2;
    if (h < heads) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const size_t p = p0 + (size_t)h * splits;
#pragma unroll
        for (int n = 0; n < NT; ++n)
            *reinterpret_cast<float2*>(a.part_o + p * HD + n * 8 + (lane & 3) * 2) = make_float2(o[n][0] * inv, o[n][1] * inv);
        if ((lane & 3) == 0) a.part_lse[p] = l == 0.f ? -INFINITY : (m == -INFINITY ? 0.f : m) + log2f(l);
    }
}

// Which range of shared keys the `range`-th is: of group g, its `split`-th of n, `per` tiles long.  `per` is the least that leaves all groups
// together no more than `ranges`, and the longest no more than there is room for; no range (n = 0) where the groups have fewer.
struct Range {
    int g, split, n, per;
};
__device__ __forceinline__ Range range_of(const Args& a, int range, int ranges) {
    const int lane = threadIdx.x & 31;
    auto tiles_of = [&](int g) {
        if (g >= a.groups) return 0;
        const int n = keys_of(a, g * a.beams), lo = a.window > 0 ? max(0, n - a.window) : 0, hi = max(lo, min(a.shared_len[g], n));
        return hi > lo ? (hi + KT - 1) / KT - lo / KT : 0;
    };
    const int first = tiles_of(lane);                      // (of 32 groups or fewer, each is read once)
    int total = first, most = first;
    for (int g = lane + 32; g < a.groups; g += 32) {
        const int n = tiles_of(g);
        total += n;
        most = max(most, n);
    }
    total = __reduce_add_sync(0xffffffffu, total);
    most = __reduce_max_sync(0xffffffffu, most);
    int per = max(1, max((total + ranges - 1) / ranges, (most + a.shared_splits - 1) / a.shared_splits));
    while (per < most) {
        int n = (first + per - 1) / per;
        for (int g = lane + 32; g < a.groups; g += 32) n += (tiles_of(g) + per - 1) / per;
        if (__reduce_add_sync(0xffffffffu, n) <= ranges) break;
        per += (per >> 3) + 1;
    }
    Range out{0, 0, 0, per};
    for (int g0 = 0, before = 0; g0 < a.groups; g0 += 32) {
        const int n = ((g0 ? tiles_of(g0 + lane) : first) + per - 1) / per;
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        const unsigned here = __ballot_sync(0xffffffffu, before + upto > range);
        if (here) {
            const int l = __ffs(here) - 1;
            out.g = g0 + l;
            out.n = __shfl_sync(0xffffffffu, n, l);
            out.split = range - (before + __shfl_sync(0xffffffffu, upto, l) - out.n);
            break;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return out;
}

// Blocks: first (range of shared keys, key head, row chunk), then a warp for (range of the row's own keys, row, key head, eight heads).
template <int RTILES, bool TMA>
__global__ void __launch_bounds__(THREADS, CTAS)
beams_kernel(const __grid_constant__ CUtensorMap map, Args a, int ranges, int chunks, int own_chunks) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    pdl_wait();
    pdl_trigger();
    const int G = a.Hq / a.Hkv, splits = a.shared_splits + a.own_splits;
    int id = blockIdx.x, from, to;
    const int n_shared = ranges * a.Hkv * chunks;
    if (id < n_shared) {
        const int chunk = id % chunks;        id /= chunks;
        const int kvh = id % a.Hkv;
        const Range x = range_of(a, id / a.Hkv, ranges);
        if (x.n == 0) return;
        shared_range(a, x.g, from, to);                    // (none where the rows do not share what they are said to)
        // ranges start at multiples of the tiles' size
        const int lo = x.split == 0 ? from : (int)min((long long)to, ((long long)(from / KT) + (long long)x.split * x.per) * KT);
        const int hi = (int)min((long long)to, ((long long)(from / KT) + (long long)(x.split + 1) * x.per) * KT);
        const int m0 = chunk * RTILES * 16, m_count = min(RTILES * 16, a.beams * G - m0);
        // the last one says of the ranges that the group does not have that they are empty
        const int empty_from = lo >= hi ? x.split : x.split + 1, empty_to = x.split + 1 == x.n ? a.shared_splits : x.split + 1;
        for (int r = threadIdx.x; r < m_count && empty_from < empty_to; r += THREADS) {
            const int b = (m0 + r) / G, h = m0 + r - b * G;
            for (int s = empty_from; s < empty_to; ++s)
                a.part_lse[((size_t)(x.g * a.beams + b) * a.Hq + kvh * G + h) * splits + s] = -INFINITY;
        }
        if (lo < hi)
            attend<RTILES, TMA>(a, &map, smem, x.g, kvh, m0, m_count, a.table + (size_t)x.g * a.beams * a.table_stride, lo, hi, x.split);
        return;
    }
    id = (id - n_shared) * WARPS + (threadIdx.x >> 5);
    const int chunk = id % own_chunks;    id /= own_chunks;
    const int kvh = id % a.Hkv;           id /= a.Hkv;
    const int split = id % a.own_splits, r = id / a.own_splits;
    if (r >= a.groups * a.beams) return;
    const int g = r / a.beams, heads = min(8, G - chunk * 8), lane = threadIdx.x & 31;
    shared_range(a, g, from, to);
    const int end = keys_of(a, r);
    const int begin = to > from ? to : (a.window > 0 ? max(0, end - a.window) : 0);
    if (split == 0) {
        // a group without a tile of shared keys has no CTA that says so
        const int n = keys_of(a, g * a.beams), lo = a.window > 0 ? max(0, n - a.window) : 0;
        if (min(a.shared_len[g], n) <= lo)
            for (int i = lane; i < heads * a.shared_splits; i += 32)
                a.part_lse[((size_t)r * a.Hq + kvh * G + chunk * 8 + i / a.shared_splits) * splits + i % a.shared_splits] = -INFINITY;
    }
    const int steps = (max(0, end - begin) + OWN_KEYS - 1) / OWN_KEYS, per = (steps + a.own_splits - 1) / a.own_splits;
    const int lo = (int)min((long long)end, begin + (long long)split * per * OWN_KEYS), hi = min(end, lo + per * OWN_KEYS);
    attend_own(a, smem, r, kvh, kvh * G + chunk * 8, heads, lo, hi, a.shared_splits + split);
}

// out[r, h, :] = sum over ranges of 2^(lse - max) part / sum of 2^(lse - max); a row without keys: zeros.  A warp a head: a lane knows one
// range's weight, and only the ranges that have keys are read.
__global__ void __launch_bounds__(128)
beams_join_kernel(const float* part_o, const float* part_lse, bf16* out, int out_stride, int Hq, int splits, int heads) {
    pdl_wait();
    const int id = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (id >= heads) return;
    const size_t p = (size_t)id * splits;
    const float lse = lane < splits ? part_lse[p + lane] : -INFINITY;
    const float M = warp_max(lse);
    float w = lse == -INFINITY ? 0.f : exp2f(lse - M);
    w /= warp_sum(w);                                      // (nothing at all: no range is read)
    constexpr int V = (HD + 127) / 128;                    // fours a lane
    float4 v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int AT_ONCE = V == 1 ? 8 : 4;                // ranges whose loads are in flight together
    for (unsigned some = __ballot_sync(0xffffffffu, lse != -INFINITY); some;) {
        float4 x[AT_ONCE][V];
        float ws[AT_ONCE];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            const int s = __ffs(some) - 1;                 // -1: none is left
            some &= some - 1;
            ws[k] = __shfl_sync(0xffffffffu, w, max(0, s));
            if (s < 0) ws[k] = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int d = lane * 4 + i * 128;
                x[k][i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (s >= 0 && d < HD) x[k][i] = *reinterpret_cast<const float4*>(part_o + (p + s) * HD + d);
            }
        }
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[i].x += ws[k] * x[k][i].x; v[i].y += ws[k] * x[k][i].y; v[i].z += ws[k] * x[k][i].z; v[i].w += ws[k] * x[k][i].w;
            }
    }
    const int r = id / Hq, h = id - r * Hq;
    bf16* to = out + (size_t)r * out_stride + (size_t)h * HD;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int d = lane * 4 + i * 128;
        if (d < HD) {
            to[d] = __float2bfloat16_rn(v[i].x);
            to[d + 1] = __float2bfloat16_rn(v[i].y);
            to[d + 2] = __float2bfloat16_rn(v[i].z);
            to[d + 3] = __float2bfloat16_rn(v[i].w);
        }
    }
}

template <int RTILES, bool TMA>
constexpr size_t smem_bytes() {
    const size_t kv = (size_t)STAGES * 2 * KT * (TMA ? HD : ROW) * sizeof(bf16) + (size_t)RTILES * 16 * ROW * sizeof(bf16) + 64;
    const size_t merge = (WARPS * 16 * (size_t)OROW + 2 * WARPS * 16) * sizeof(float), own = (size_t)WARPS * OWN_STAGES * 2 * OWN_KEYS * ROW * sizeof(bf16);
    return 1024 /*alignment*/ + (kv > merge ? (kv > own ? kv : own) : (merge > own ? merge : own));
}

// One layer of the cache, [page][K|V][kv head][slot][HD], seen as a matrix of HD-wide rows, in boxes of 64 columns x box_rows rows with the
// 128-byte swizzle.
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
int cache_map(const void* ptr, long long rows, int box_rows, CUtensorMap* out) {
    static std::mutex mu;
    static EncodeTiledFn fn = nullptr;
    {
        std::lock_guard<std::mutex> lock(mu);
        if (!fn) {
            void* sym = nullptr;
            cudaDriverEntryPointQueryResult q;
            if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
                return (int)cudaErrorNotSupported;
            fn = reinterpret_cast<EncodeTiledFn>(sym);
        }
    }
    cuuint64_t dims[2] = {(cuuint64_t)HD, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)HD * 2};
    cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, elem[2] = {1, 1};
    return fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? 0
               : (int)cudaErrorInvalidValue;
}

template <int RTILES, bool TMA>
int run(Args a, long long pages, cudaStream_t stream) {
    constexpr int bytes = (int)smem_bytes<RTILES, TMA>();
    static unsigned long long configured = 0;              // devices, a bit each (one that is set twice is set to the same)
    int device = 0;
    RI_CHECKED((int)cudaGetDevice(&device));
    if (device > 63 || !(configured >> device & 1)) {
        RI_CHECKED((int)cudaFuncSetAttribute(beams_kernel<RTILES, TMA>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        if (device <= 63) configured |= 1ull << device;
    }
    CUtensorMap map = {};
    if constexpr (TMA) {
        a.box_rows = a.page_size < KT ? a.page_size : KT;
        RI_CHECKED(cache_map(a.cache, pages * 2 * a.Hkv * a.page_size, a.box_rows, &map));
    }
    const int G = a.Hq / a.Hkv, chunks = (a.beams * G + RTILES * 16 - 1) / (RTILES * 16), own_chunks = (G + 7) / 8;
    const long long units = (long long)a.groups * a.beams * a.Hkv * own_chunks * a.own_splits;
    // ranges of shared keys: as many as make `target` CTAs, and one a group at least
    const int made = a.target / (a.Hkv * chunks), ranges = made > a.groups ? made : a.groups;
    const long long blocks = (long long)ranges * a.Hkv * chunks + (units + WARPS - 1) / WARPS;
    if (blocks * WARPS > 0x7fffffffll) return (int)cudaErrorInvalidValue;
    return ri_launch(beams_kernel<RTILES, TMA>, dim3((unsigned)blocks), dim3(THREADS), (size_t)bytes, stream, map, a, ranges, chunks, own_chunks);
}
bool by_tma(const void* cache, int page_size, long long pages, int Hkv) {
    return BY_TMA && (page_size == 8 || page_size == 16 || page_size == 32 || page_size % 64 == 0) && (reinterpret_cast<uintptr_t>(cache) & 15) == 0 &&
           (pages + 1) * 2 * Hkv * page_size < (1ll << 31);     // rows are 32-bit coordinates
}
template <bool TMA>
int run_rows(const Args& a, long long pages, cudaStream_t s) {
    const int rows = a.beams * (a.Hq / a.Hkv);
    return rows <= 16 ? run<1, TMA>(a, pages, s) : rows <= 32 ? run<2, TMA>(a, pages, s) : run<4, TMA>(a, pages, s);
}
}  // namespace

// Row tiles of 16 a CTA takes of a group's beams x heads
RI_API int ri_attention_beams_row_tiles(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }
RI_API int ri_attention_beams_ctas_per_sm() { return CTAS; }

// part_o: rows * Hq * (shared_splits + own_splits) * HD floats, part_lse the same without HD.  `error` gets 22 where a wait for a copy ran out.
RI_API int ri_attention_beams(const void* q, int q_stride, void* out, int out_stride, const void* cache, long long pages, const int* table,
                              int table_stride, int table_cols, const int* kv_len, const int* shared_len, int groups, int beams, int Hq, int Hkv,
                              int page_size, float scale, int window, int shared_splits, int own_splits, int target, float* part_o, float* part_lse,
                              int* error, void* stream) {
    if (groups <= 0) return 0;
    if (beams < 1 || beams > MAX_BEAMS || Hkv <= 0 || Hq % Hkv != 0 || page_size < 1 || shared_splits < 1 || own_splits < 1 ||
        shared_splits + own_splits > 32 || !part_o || !part_lse || !error || (long long)groups * beams * Hq > 0x7fffffffll)
        return (int)cudaErrorInvalidValue;
    const Args a{(const bf16*)q, q_stride, (const bf16*)cache, table, table_stride, (int)min((long long)table_cols * page_size, 0x7fffffffll - 256),
                 (int)min(pages, 0x7fffffffll), kv_len, shared_len, beams, Hq, Hkv, page_size, scale * 1.4426950408889634f, window, groups, shared_splits, own_splits,
                 target < 1 ? 1 : target, part_o, part_lse, error, 8};
    cudaStream_t s = (cudaStream_t)stream;
    bool tma = false;
    if constexpr (BY_TMA) {
        tma = by_tma(cache, page_size, pages, Hkv);
        if (tma) RI_CHECKED(run_rows<true>(a, pages, s));
    }
    if (!tma) RI_CHECKED(run_rows<false>(a, pages, s));
    const int heads = groups * beams * Hq;
    RI_CHECKED(ri_launch(beams_join_kernel, dim3((heads + 3) / 4), dim3(128), 0, s, part_o, part_lse, (bf16*)out, out_stride, Hq,
                         shared_splits + own_splits, heads));
    return ri_launch_status();
}

RI_API void ri_set_pdl(int on) { ri_pdl_flag() = on ? 1 : 0; }
