// Attention of a step of single tokens whose rows are the beams of requests: the beams of a request share the keys of their prompt and have
// some of their own.  bf16, paged, grouped-query, compiled for one RI_HEAD_DIM (a multiple of 16, at most 256).
//
//     out[r, h] = sum_k softmax_k(scale q[r, h] . K[k]) V[k],   k over [kv_len[r] - window, kv_len[r])
//
// Keys before shared_len[g] are the same for every row of group g, whose rows follow one another: one CTA reads a range of them, by the
// first row's table, for all beams x heads of a key head, which are the M dimension of the matrix products.  Keys from there on are read
// by each row's own table.  Both leave partial results (a sum weighted by 2^(score - maximum), its log-sum-exp in base 2) that a second
// kernel joins.  RustInfer's decode attention reads a request's keys for that request alone
// (crates/infer-backend-cuda/src/kernels/flash_attn_gqa/flash_attn_paged_decode.cu:75-340).
//
// What bounds it is the cache's stream: shared keys and values once a request, the beams' own once a beam.  Scores, maxima, sums and
// outputs are 32-bit.  A weight enters the product with the values as two bf16 pieces that add up to it to 2^-17 of itself: rounded to one
// piece it would be off by up to 2^-9, as much as the stored output's own rounding.
#include "common.cuh"

#ifndef RI_HEAD_DIM
#error "compile with -DRI_HEAD_DIM=<head size>"
#endif

namespace {
constexpr int HD = RI_HEAD_DIM;
static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "beam attention: head size multiple of 16, at most 256");
constexpr int KT = 64;                                     // keys a tile
constexpr int ROW = HD + 8;                                // padded rows: 16 bytes on, ldmatrix meets no bank twice
constexpr int CH = HD / 8;                                 // 16-byte pieces a row
constexpr int KS = HD / 16;
constexpr int NT = HD / 8;
constexpr int WARPS = 4;
constexpr int THREADS = 32 * WARPS;
constexpr int STAGES = HD <= 128 ? 3 : 2;
constexpr int MAX_BEAMS = 64;

__device__ __forceinline__ void cp_async16(void* smem, const void* gmem, bool valid) {
    const unsigned s = (unsigned)__cvta_generic_to_shared(smem);
    const int n = valid ? 16 : 0;                          // 0 bytes read: the 16 bytes are filled with zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(s), "l"(gmem), "r"(n));
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N)); }
__device__ __forceinline__ void ldmatrix_x4(unsigned (&r)[4], const void* p) {
    const unsigned s = (unsigned)__cvta_generic_to_shared(p);
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s));
}
__device__ __forceinline__ void ldmatrix_x4_trans(unsigned (&r)[4], const void* p) {
    const unsigned s = (unsigned)__cvta_generic_to_shared(p);
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
    const int* kv_len;
    const int* shared_len;
    int beams, Hq, Hkv, page_size;
    float scale_log2;
    int window, shared_splits, own_splits;
    float* part_o;
    float* part_lse;
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

// Keys [lo, hi) by table row `bt` for the rows m0 .. m0 + m_count - 1 (of beams x heads) of group g, RTILES tiles of 16 rows in one CTA.
template <int RTILES>
__device__ __forceinline__ void attend(const Args& a, unsigned char* smem, int g, int kvh, int m0, int m_count, const int* bt, int lo, int hi, int part) {
    constexpr int KG = WARPS / RTILES;                     // warps that share a row tile take parts of a tile's keys
    constexpr int WK = KT / KG;                            // keys a warp takes of a tile
    constexpr int NK = WK / 8;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = a.Hq / a.Hkv, splits = a.shared_splits + a.own_splits;
    bf16* Qs = reinterpret_cast<bf16*>(smem);              // [RTILES * 16][ROW]
    bf16* KVs = Qs + RTILES * 16 * ROW;                    // [STAGES][K | V][KT][ROW]
    const int rt = warp / KG, kg = warp % KG;

    for (int c = tid; c < RTILES * 16 * CH; c += THREADS) {
        const int r = c / CH, ch = c - r * CH, m = m0 + r;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (r < m_count) {
            const int b = m / G, h = m - b * G;
            v = *reinterpret_cast<const uint4*>(a.q + (size_t)(g * a.beams + b) * a.q_stride + (size_t)(kvh * G + h) * HD + ch * 8);
        }
        *reinterpret_cast<uint4*>(Qs + r * ROW + ch * 8) = v;
    }
    const size_t head_step = (size_t)a.page_size * HD;
    const int shift = (a.page_size & (a.page_size - 1)) == 0 ? __ffs(a.page_size) - 1 : -1;
    auto load = [&](int k0, int stage) {
        bf16* Ks = KVs + (size_t)stage * 2 * KT * ROW;
        bf16* Vs = Ks + KT * ROW;
        for (int c = tid; c < KT * CH; c += THREADS) {
            const int kk = c / CH, ch = c - kk * CH, key = k0 + kk;
            const bool ok = key < hi;
            const bf16 *sk = a.cache, *sv = a.cache;
            if (ok) {
                const int blk = shift >= 0 ? key >> shift : key / a.page_size;
                const int off = key - blk * a.page_size;
                sk = a.cache + ((size_t)bt[blk] * 2 * a.Hkv + kvh) * head_step + (size_t)off * HD + ch * 8;
                sv = sk + (size_t)a.Hkv * head_step;
            }
            cp_async16(Ks + kk * ROW + ch * 8, sk, ok);
            cp_async16(Vs + kk * ROW + ch * 8, sv, ok);
        }
    };
    const int tiles = hi > lo ? (hi - lo + KT - 1) / KT : 0;
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
        if (s < tiles) load(lo + s * KT, s);
        cp_async_commit();
    }
    __syncthreads();
    unsigned qf[KS][4];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) ldmatrix_x4(qf[ks], Qs + (rt * 16 + (lane & 15)) * ROW + ks * 16 + (lane >> 4) * 8);
    float o[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    for (int t = 0; t < tiles; ++t) {
        cp_async_wait<STAGES - 2>();
        __syncthreads();                                   // the tile has come, and the one before it is used up
        if (t + STAGES - 1 < tiles) load(lo + (t + STAGES - 1) * KT, (t + STAGES - 1) % STAGES);
        cp_async_commit();
        const bf16* Ks = KVs + (size_t)(t % STAGES) * 2 * KT * ROW;
        const bf16* Vs = Ks + KT * ROW;
        const int kw0 = kg * WK, key0 = lo + t * KT + kw0;
        if (key0 >= hi) continue;
        float s[NK][4];
#pragma unroll
        for (int n = 0; n < NK; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int n2 = 0; n2 < NK / 2; ++n2) {
                unsigned kf[4];
                ldmatrix_x4(kf, Ks + (kw0 + n2 * 16 + (lane & 7) + (lane >> 4) * 8) * ROW + ks * 16 + ((lane >> 3) & 1) * 8);
                mma_bf16(s[2 * n2], qf[ks], kf[0], kf[1]);
                mma_bf16(s[2 * n2 + 1], qf[ks], kf[2], kf[3]);
            }
        float mx[2] = {-INFINITY, -INFINITY};
        const int left = hi - key0;                        // keys of this warp's that exist
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[n][e] = n * 8 + (lane & 3) * 2 + (e & 1) < left ? s[n][e] * a.scale_log2 : -INFINITY;
                mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
            }
        float alpha[2], muse[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
            const float mnew = fmaxf(m[i], mx[i]);
            muse[i] = mnew == -INFINITY ? 0.f : mnew;
            alpha[i] = exp2f(m[i] - muse[i]);
            m[i] = mnew;
            l[i] *= alpha[i];
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            o[n][0] *= alpha[0]; o[n][1] *= alpha[0];
            o[n][2] *= alpha[1]; o[n][3] *= alpha[1];
        }
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[n][e] = exp2f(s[n][e] - muse[e >> 1]);
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
                ldmatrix_x4_trans(vf, Vs + (kw0 + n2 * 16 + (lane & 15)) * ROW + np * 16 + (lane >> 4) * 8);
                mma_bf16(o[2 * np], ph, vf[0], vf[1]);
                mma_bf16(o[2 * np + 1], ph, vf[2], vf[3]);
                mma_bf16(o[2 * np], pl, vf[0], vf[1]);
                mma_bf16(o[2 * np + 1], pl, vf[2], vf[3]);
            }
        }
    }
    cp_async_wait<0>();
    __syncthreads();

    // the warps' states through shared memory (the tiles are used up)
    float* Os = reinterpret_cast<float*>(KVs);             // [WARPS][16][HD]
    float* Ms = Os + WARPS * 16 * HD;                      // [WARPS][16]
    float* Ls = Ms + WARPS * 16;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        const int r = (lane >> 2) + 8 * i;
        float* orow = Os + ((size_t)warp * 16 + r) * HD + (lane & 3) * 2;
#pragma unroll
        for (int n = 0; n < NT; ++n) *reinterpret_cast<float2*>(orow + n * 8) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
        if ((lane & 3) == 0) { Ms[warp * 16 + r] = m[i]; Ls[warp * 16 + r] = l[i]; }
    }
    __syncthreads();
    for (int idx = tid; idx < m_count * HD; idx += THREADS) {
        const int r = idx / HD, d = idx - r * HD, w0 = (r >> 4) * KG, rr = r & 15;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < KG; ++w) M = fmaxf(M, Ms[(w0 + w) * 16 + rr]);
        float L = 0.f, O = 0.f;
        const float muse = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int w = 0; w < KG; ++w) {
            const float f = exp2f(Ms[(w0 + w) * 16 + rr] - muse);
            L += Ls[(w0 + w) * 16 + rr] == 0.f ? 0.f : Ls[(w0 + w) * 16 + rr] * f;
            O += Ls[(w0 + w) * 16 + rr] == 0.f ? 0.f : Os[((size_t)(w0 + w) * 16 + rr) * HD + d] * f;
        }
        const int mm = m0 + r, b = mm / G, h = mm - b * G;
        const size_t p = ((size_t)(g * a.beams + b) * a.Hq + kvh * G + h) * splits + part;
        a.part_o[p * HD + d] = L == 0.f ? 0.f : O / L;
        if (d == 0) a.part_lse[p] = L == 0.f ? -INFINITY : muse + log2f(L);      // what is no number stays none
    }
}

// Blocks: first (group, key head, row chunk, range of shared keys), then (row, key head, head chunk, range of the row's own keys).
template <int RTILES>
__global__ void __launch_bounds__(THREADS)
beams_kernel(Args a, int groups, int chunks, int own_chunks) {
    extern __shared__ __align__(16) unsigned char smem[];
    pdl_wait();
    pdl_trigger();
    const int G = a.Hq / a.Hkv;
    int id = blockIdx.x, from, to;
    const int n_shared = groups * a.Hkv * chunks * a.shared_splits;
    if (id < n_shared) {
        const int split = id % a.shared_splits;  id /= a.shared_splits;
        const int chunk = id % chunks;           id /= chunks;
        const int kvh = id % a.Hkv, g = id / a.Hkv;
        shared_range(a, g, from, to);
        const int tiles = (to - from + KT - 1) / KT, per = (tiles + a.shared_splits - 1) / a.shared_splits;
        const int lo = min(to, from + split * per * KT), hi = min(to, lo + per * KT);
        const int m0 = chunk * RTILES * 16;
        attend<RTILES>(a, smem, g, kvh, m0, min(RTILES * 16, a.beams * G - m0), a.table + (size_t)g * a.beams * a.table_stride, lo, hi, split);
        return;
    }
    id -= n_shared;
    const int split = id % a.own_splits;  id /= a.own_splits;
    const int chunk = id % own_chunks;    id /= own_chunks;
    const int kvh = id % a.Hkv, r = id / a.Hkv, g = r / a.beams, b = r - g * a.beams;
    shared_range(a, g, from, to);
    const int end = keys_of(a, r);
    const int begin = to > from ? to : (a.window > 0 ? max(0, end - a.window) : 0);
    const int tiles = (max(0, end - begin) + KT - 1) / KT, per = (tiles + a.own_splits - 1) / a.own_splits;
    const int lo = min(end, begin + split * per * KT), hi = min(end, lo + per * KT);
    attend<1>(a, smem, g, kvh, b * G + chunk * 16, min(16, G - chunk * 16), a.table + (size_t)r * a.table_stride, lo, hi, a.shared_splits + split);
}

// out[r, h, :] = sum over ranges of 2^(lse - max) part / sum of 2^(lse - max); a row without keys: zeros
__global__ void beams_join_kernel(const float* part_o, const float* part_lse, bf16* out, int out_stride, int Hq,
                                  int splits) {
    pdl_wait();
    const int r = blockIdx.x, h = blockIdx.y;
    const size_t p = ((size_t)r * Hq + h) * splits;
    float M = -INFINITY;
    for (int s = 0; s < splits; ++s) M = fmaxf(M, part_lse[p + s]);
    for (int d = threadIdx.x; d < HD; d += blockDim.x) {
        float W = 0.f, O = 0.f;
        for (int s = 0; s < splits; ++s) {
            const float lse = part_lse[p + s];
            if (lse == -INFINITY) continue;                // a range without keys
            const float w = exp2f(lse - M);
            W += w;
            O += w * part_o[(p + s) * HD + d];
        }
        out[(size_t)r * out_stride + (size_t)h * HD + d] = __float2bfloat16_rn(W == 0.f ? 0.f : O / W);
    }
}

constexpr size_t smem_bytes(int rtiles) {
    const size_t kv = (size_t)STAGES * 2 * KT * ROW * sizeof(bf16), merge = (WARPS * 16 * (size_t)HD + 2 * WARPS * 16) * sizeof(float);
    return (size_t)rtiles * 16 * ROW * sizeof(bf16) + (kv > merge ? kv : merge);
}
template <int RTILES>
int run(const Args& a, int groups, cudaStream_t stream) {
    static int configured = -1;
    if (configured != 0) {
        configured = (int)cudaFuncSetAttribute(beams_kernel<RTILES>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes(RTILES));
        if (configured != 0) return configured;
    }
    const int G = a.Hq / a.Hkv, chunks = (a.beams * G + RTILES * 16 - 1) / (RTILES * 16), own_chunks = (G + 15) / 16;
    const long long blocks = (long long)groups * a.Hkv * ((long long)chunks * a.shared_splits + (long long)a.beams * own_chunks * a.own_splits);
    if (blocks > 0x7fffffffll) return (int)cudaErrorInvalidValue;
    return ri_launch(beams_kernel<RTILES>, dim3((unsigned)blocks), dim3(THREADS), smem_bytes(RTILES), stream, a, groups, chunks, own_chunks);
}
}  // namespace

// Row tiles of 16 a CTA takes of a group's beams x heads
RI_API int ri_attention_beams_row_tiles(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }
RI_API int ri_attention_beams_ctas_per_sm(int row_tiles) {
    const int n = (int)(227 * 1024 / (smem_bytes(row_tiles) + 1024));
    return n < 1 ? 1 : n < 2048 / THREADS ? n : 2048 / THREADS;
}

// part_o: rows * Hq * (shared_splits + own_splits) * HD floats, part_lse the same without HD.
RI_API int ri_attention_beams(const void* q, int q_stride, void* out, int out_stride, const void* cache, const int* table, int table_stride, int table_cols,
                              const int* kv_len, const int* shared_len, int groups, int beams, int Hq, int Hkv, int page_size, float scale,
                              int window, int shared_splits, int own_splits, float* part_o, float* part_lse, void* stream) {
    if (groups <= 0) return 0;
    if (beams < 1 || beams > MAX_BEAMS || Hkv <= 0 || Hq % Hkv != 0 || Hq > 65535 || page_size < 1 || shared_splits < 1 || own_splits < 1 || !part_o ||
        !part_lse)
        return (int)cudaErrorInvalidValue;
    const Args a{(const bf16*)q, q_stride, (const bf16*)cache, table, table_stride,
                 (int)min((long long)table_cols * page_size, 0x7fffffffll - KT), kv_len, shared_len, beams, Hq, Hkv, page_size,
                 scale * 1.4426950408889634f, window, shared_splits, own_splits, part_o, part_lse};
    cudaStream_t s = (cudaStream_t)stream;
    const int tiles = ri_attention_beams_row_tiles(beams * (Hq / Hkv));
    RI_CHECKED(tiles == 1 ? run<1>(a, groups, s) : tiles == 2 ? run<2>(a, groups, s) : run<4>(a, groups, s));
    RI_CHECKED(ri_launch(beams_join_kernel, dim3(groups * beams, Hq), dim3(HD < 128 ? 64 : 128), 0, s, part_o, part_lse, (bf16*)out, out_stride, Hq,
                         shared_splits + own_splits));
    return ri_launch_status();
}

RI_API void ri_set_pdl(int on) { ri_pdl_flag() = on ? 1 : 0; }
