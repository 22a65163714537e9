// Beam search's choice: of every group of `beams` rows the `picks` best continuations by
//
//     score(b, t) = scores[b] + x[b, t] - log sum_t' exp x[b, t']
//
// in descending order, equal scores by ascending (row, token).  RustInfer chooses one token a request
// (crates/infer-worker/src/application/sampler_stack.rs:242-351) and has no counterpart.
//
// Within a row a score falls with its logit, so the row's own best `picks` logits are all that can be chosen, and the
// logits are read once: a CTA walks a slice of a row, keeps the sum of its weights and what may be among the slice's best.
// These two are all that leaves the CTA; a second kernel, a CTA a group, puts the slices' sums together in 64
// bits, scores what the slices sent in 64 bits and orders it.
//
// The best `picks` of a slice without a sort: let t be a value that at least `picks` threads' own maxima reach; then at
// least `picks` elements reach it and nothing below it is among the best.  t is found by bisection on the maxima, a
// barrier with a count a step, and stops as soon as no more than one and a half times `picks` threads are left.  The few elements
// that reach t leave the CTA as they come; in a slice of several chunks they are found by each thread's maximum of every chunk,
// and those few chunks are read once more (from L2).  Where more than twice `picks` do, a warp counts the ones ahead of
// each, which is its rank, and the best `picks` leave.  Where more than the gathering's room reach t (thousands of equal logits,
// words that are forbidden), the last element that belongs is found exactly, by bisection over values and then over indices.
// The second kernel does the same with 64-bit scores.
//
// Scores and the sums over slices are 64-bit: the rows of a group compete through the sums, and a choice hangs on
// differences however small.  Weights are 32-bit exponentials, summed in 32 bits over a thread's sixteen of a chunk and in 64 from there.
#include "common.cuh"

namespace {
constexpr int ST = 256;                                    // threads of a slice
constexpr int NV = 4;                                      // 16-byte loads of a thread a chunk
constexpr int CTAS = 4;                                    // CTAs an SM, which walk over slices
constexpr int STAGES = 2;                                  // chunks of a slice in shared memory
// (512 rows of 128,256 logits, 48 picks of 16 beams, slices of 8 chunks, us a call: 4 CTAs and 2 stages 69, 3 and 3 73, 3 and 2 70; 512 threads, 2 and 2 73; chunks of
// half the size 81.  The logits' stream with its sums alone takes 48)
constexpr int MAX_CHUNKS = 16;                             // chunks of a slice
constexpr int AGAIN = 2048;                                // threads' chunks that may be read once more
constexpr int LISTS = 1024;                                // slices of a group whose sums are kept in shared memory
constexpr int MT = 512;                                    // threads of a group
constexpr int PLACES = 8192;                               // of a group's pool that shared memory holds
constexpr int CAP = 1024;                                  // room of the gathering
constexpr int MAX_PICKS = 128, MAX_BEAMS = 64;

__device__ __forceinline__ unsigned ordered(float v) {     // ascending with v; -inf is 0x007fffff, so 0 is below every value
    const unsigned u = __float_as_uint(v);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
// of a logit: both zeros are one value
__device__ __forceinline__ unsigned key_of(float x) { return ordered(x + 0.f); }
__device__ __forceinline__ float from_ordered(unsigned k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

constexpr float L = 1.4426950408889634f;                   // log2 e in 32 bits
// A slice's sum of weights, its largest logit, and how many of its elements left the CTA.  The weights are 2^(x L - ref) with
// ref = ceil(m L), or exp(x - m) where `by_difference`
struct SliceStat {
    double sum;
    float m;
    int n;
};
__device__ __forceinline__ bool by_difference(float m) { return !(fabsf(m) <= 65536.f); }      // beyond, x L - ref is not near enough
__device__ __forceinline__ float whole_ref(float m) { return ceilf(m * L); }
constexpr float LEAST_REF = -131072.f;                     // below whole_ref(-65536) = -94548
__device__ __forceinline__ float two_to(float whole) {     // 2^whole for a whole number up to 0, exactly; 0 below the normal numbers
    return whole < -126.f ? 0.f : __int_as_float((127 + (int)whole) << 23);
}
__device__ __forceinline__ float ex2(float x) {            // 2 ulp
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// count of a block's elements (each thread brings its own)
__device__ __forceinline__ int block_count(int mine, int* cell) {
    const int w = __reduce_add_sync(0xffffffffu, mine);
    __syncthreads();
    if (threadIdx.x == 0) *cell = 0;
    __syncthreads();
    if ((threadIdx.x & 31) == 0 && w) atomicAdd(cell, w);
    __syncthreads();
    return *cell;
}

// A value that at least `picks` of the threads' maxima reach, by bisection on the ordered bits; `top` is the largest.
// Needs at least `picks` threads whose `mine` is at least `floor`.
__device__ __forceinline__ unsigned reach(unsigned mine, unsigned floor, unsigned top, int picks) {
    unsigned lo = floor, hi = top;                         // count(>= lo) >= picks
    while (lo < hi) {
        const unsigned mid = lo + (hi - lo + 1) / 2;       // in (lo, hi]
        const int n = __syncthreads_count(mine >= mid);
        if (n >= picks) {
            lo = mid;
            if (2 * n <= 3 * picks) break;
        } else {
            hi = mid - 1;
        }
    }
    return lo;
}

__device__ __forceinline__ void copy_async16(unsigned to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_async4(unsigned to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_async8(unsigned to, const void* from, bool there) {       // else zeros
    const int n = there ? 8 : 0;
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;\n" ::"r"(to), "l"(from), "r"(n) : "memory");
}

__global__ void __launch_bounds__(ST, CTAS)
beam_slices_kernel(const float* logits, long long ld, int vocab, const float* scores, int picks, int items, int slices,
                   int vectors_a_slice, unsigned long long* best, SliceStat* stat) {
    extern __shared__ float4 ring[];                       // [STAGES][NV][W][33]: a warp reads what it has fetched itself, so no barrier
    __shared__ unsigned long long list[CAP];
    __shared__ unsigned red_hi[ST / 32], red_lo[ST / 32];
    __shared__ double wsum[ST / 32];
    __shared__ bf16 tops[MAX_CHUNKS][ST];                       // rounded up
    __shared__ unsigned short again[AGAIN];
    __shared__ int cell, listed;
    constexpr int W = ST / 32, CHUNK = NV * ST;
    constexpr unsigned MINUS_INF = 0x007fffffu;            // ordered(-inf)
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();
    pdl_trigger();
    struct Slice {                                         // of row r, vectors v0 .. v1 - 1, elements up to e_hi
        const float* row;
        int v0, v1, e_hi, shift;                           // the row starts `shift` elements behind a 16-byte boundary
        bool dead;
    } now, then;
    auto open = [&](Slice& s, int item) {
        const int r = item / slices;
        s.row = logits + (size_t)r * ld;
        s.v0 = (item - r * slices) * vectors_a_slice;
        s.v1 = min(s.v0 + vectors_a_slice, (vocab + 3) >> 2);
        s.e_hi = min(vocab, 4 * s.v1);
        s.shift = (int)((reinterpret_cast<uintptr_t>(s.row) >> 2) & 3);
        s.dead = !(scores[r] > -INFINITY);                 // without a future: not read
    };
    // A vector of the ring holds 16 aligned bytes: where the row starts `shift` elements behind a boundary, a thread's four elements lie in
    // its own and in the next lane's, and the warp fetches a 33rd.
    const unsigned mine_at = (unsigned)__cvta_generic_to_shared(ring) + (warp * 33 + lane) * 16;
    constexpr unsigned STEP = W * 33 * 16, STAGE = NV * STEP;      // bytes from a thread's vector to its next, and to the next stage
    auto fetch = [&](const Slice& s, int v, int stage) {
        const int e0 = 4 * v - s.shift;                    // the chunk's first element
        if (v < s.v1 && !s.dead) {
            const unsigned to = mine_at + stage * STAGE;
            if (e0 >= 0 && e0 + 4 * CHUNK + (s.shift ? 4 : 0) <= s.e_hi) {             // all of it lies in the slice
                const float* from = s.row + e0 + 4 * tid;
#pragma unroll
                for (int i = 0; i < NV; ++i) copy_async16(to + i * STEP, from + i * (4 * ST));
                if (s.shift && lane == 0) {
#pragma unroll
                    for (int i = 0; i < NV; ++i) copy_async16(to + i * STEP + 32 * 16, from + i * (4 * ST) + 4 * 32);
                }
            } else {
#pragma unroll 1
                for (int i = 0; i < NV; ++i)
#pragma unroll 1
                    for (int j = lane; j < 32 + (s.shift != 0); j += 32) {
                        const int e = e0 + 4 * (i * ST + warp * 32 + j);
                        const unsigned at = to + i * STEP + (j - lane) * 16;
                        if (e >= 0 && e + 4 <= s.e_hi) {
                            copy_async16(at, s.row + e);
                        } else {
                            for (int k = 0; k < 4; ++k)
                                if (e + k >= 0 && e + k < s.e_hi) copy_async4(at + 4 * k, s.row + e + k);
                                else asm volatile("st.shared.f32 [%0], %1;" ::"r"(at + 4 * k), "f"(-INFINITY) : "memory");
                        }
                    }
            }
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    };
    auto prime = [&](const Slice& s) {
#pragma unroll
        for (int c = 0; c < STAGES - 1; ++c) fetch(s, s.v0 + c * CHUNK, c);
    };
    if ((int)blockIdx.x < items) {
        open(then, blockIdx.x);
        prime(then);
    }
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
    now = then;
    const float* const row = now.row;
    const int v0 = now.v0, v1 = now.v1, e_lo = 4 * v0, e_hi = now.e_hi, count = max(0, e_hi - e_lo);
    unsigned long long* const mine_best = best + (size_t)item * (2 * picks);
    SliceStat* const mine_stat = stat + item;
    __syncthreads();                                       // the slice before is done with what the block shares
    if (tid == 0) cell = listed = 0;
    auto next = [&]() {
        if (item + (int)gridDim.x < items) {
            open(then, item + gridDim.x);
            prime(then);                                   // on its way while this slice's end is made
        }
    };
    if (now.dead) {                                        // every score -inf, by index
        for (int i = tid; i < min(picks, count); i += ST) mine_best[i] = ((unsigned long long)MINUS_INF << 32) | (unsigned)(0xffffffffu - (unsigned)(e_lo + i));
        if (tid == 0) *mine_stat = SliceStat{0.0, -INFINITY, min(picks, count)};
        next();
        continue;
    }
    // A thread's sum of 2^(x L - ref), L = log2 e in 32 bits, ref a whole number that is at least the thread's largest x L: one fused
    // multiply-add an element, whose own rounding is all that is lost, and moving on to another ref is exact.  A chunk's sixteen are
    // added up in 32 bits, the rest in 64.  A ref starts below every one that a slice summed so can have (whole_ref(m) > LEAST_REF): words masked by
    // large finite numbers weigh nothing beside it, where a ref of their own, rounded by more than the exponents' range, would give them any weight.
    double sum = 0.0;
    float ref = LEAST_REF, top = -INFINITY;                // (top: what is no number does not count)
    auto add_up = [&](const float (&x)[4 * NV], float high) {
        const float to = fmaxf(ref, ceilf(high * L));
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4 * NV; ++i) part[i & 3] += ex2(fmaf(x[i], L, -to));
        sum = sum * (double)ex2(ref - to) + (double)((part[0] + part[1]) + (part[2] + part[3]));
        ref = to;
    };
    auto highest = [&](const float (&x)[4 * NV]) {
        float h[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 4 * NV; ++i) h[i & 3] = fmaxf(h[i & 3], x[i]);
        return fmaxf(fmaxf(h[0], h[1]), fmaxf(h[2], h[3]));
    };
    unsigned t = 0;                                        // a value that the slice's best all reach (0: all do)
    float tf = -INFINITY;
    auto gather = [&](const float (&x)[4 * NV], int v) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (!(fmaxf(fmaxf(x[4 * i], x[4 * i + 1]), fmaxf(x[4 * i + 2], x[4 * i + 3])) < tf)) {
                const int e = 4 * (v + i * ST + tid);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const unsigned o = key_of(fmaxf(x[4 * i + k], -INFINITY));               // what is no number ranks with -inf
                    if (o >= t && e + k < e_hi) {
                        const int at = atomicAdd(&listed, 1);
                        if (at < CAP) list[at] = ((unsigned long long)o << 32) | (unsigned)(0xffffffffu - (unsigned)(e + k));
                    }
                }
            }
    };
    auto block_high = [&](unsigned mine) -> unsigned {
        const unsigned h = __reduce_max_sync(0xffffffffu, mine);
        __syncthreads();
        if (lane == 0) red_hi[warp] = h;
        __syncthreads();
        return __reduce_max_sync(0xffffffffu, red_hi[lane & (W - 1)]);
    };

    // An element's thread goes by its index alone, whatever the row's alignment: equal rows get equal sums, and their continuations
    // are equals that go by index.
    float x[4 * NV];
    for (int v = v0, chunk = 0, stage = 0; v < v1; v += CHUNK, ++chunk, stage = stage + 1 == STAGES ? 0 : stage + 1) {
        fetch(now, v + (STAGES - 1) * CHUNK, stage == 0 ? STAGES - 1 : stage - 1);
        asm volatile("cp.async.wait_group %0;\n" ::"n"(STAGES - 1) : "memory");
        __syncwarp();
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const float4* const from = ring + ((stage * NV + i) * W + warp) * 33 + lane;
            float4 f = from[0];
            if (now.shift) {
                const float4 g = from[1];
                f = now.shift == 1 ? make_float4(f.y, f.z, f.w, g.x) : now.shift == 2 ? make_float4(f.z, f.w, g.x, g.y) : make_float4(f.w, g.x, g.y, g.z);
            }
            x[4 * i] = f.x; x[4 * i + 1] = f.y; x[4 * i + 2] = f.z; x[4 * i + 3] = f.w;
        }
        __syncwarp();                                      // the stage is free
        const float high = highest(x);
        top = fmaxf(top, high);
        tops[chunk][tid] = __float2bfloat16_ru(high);
        add_up(x, high);
    }
    next();
    const unsigned own = key_of(top);
    const int holders = min(ST, v1 - v0);                  // threads with an element of the slice
    {
        const unsigned lo = __reduce_min_sync(0xffffffffu, tid < holders ? own : 0xffffffffu);
        if (lane == 0) red_lo[warp] = lo;
    }
    const unsigned key_m = block_high(own);
    const float m = from_ordered(key_m);
    if (count > 2 * picks) {
        t = reach(own, holders >= picks ? __reduce_min_sync(0xffffffffu, red_lo[lane & (W - 1)]) : MINUS_INF, key_m, picks);
        tf = from_ordered(t);
    }
    if (v1 - v0 <= CHUNK) {
        if (own >= t) gather(x, v0);
    } else {
        // the few chunks of a thread in which something reaches t are read once more, a thread a vector
        for (int c = 0, v = v0; v < v1; ++c, v += CHUNK)
            if (__bfloat162float(tops[c][tid]) >= tf) {
                const int to = atomicAdd(&cell, 1);
                if (to < AGAIN) again[to] = (unsigned short)(c * ST + tid);
            }
        __syncthreads();
        const bool fits = cell <= AGAIN;                   // else more elements than the gathering has room for
        if (!fits && tid == 0) listed = CAP + 1;
        const int vectors = fits ? cell * NV : 0;
        constexpr int AT_ONCE = 2;                         // vectors in flight together
        for (int i0 = tid; i0 < vectors; i0 += AT_ONCE * ST) {
            float y[AT_ONCE][4];
            int e[AT_ONCE];
#pragma unroll
            for (int q = 0; q < AT_ONCE; ++q) {
                const int i = i0 + q * ST;
                e[q] = e_hi;
                if (i < vectors) {
                    const int at = again[i / NV], c = at / ST;
                    e[q] = 4 * (v0 + c * CHUNK + (i & (NV - 1)) * ST + (at & (ST - 1)));
                }
                if (now.shift == 0 && e[q] + 4 <= e_hi) {
                    const float4 f = *reinterpret_cast<const float4*>(row + e[q]);
                    y[q][0] = f.x; y[q][1] = f.y; y[q][2] = f.z; y[q][3] = f.w;
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) y[q][k] = e[q] + k < e_hi ? row[e[q] + k] : -INFINITY;
                }
            }
#pragma unroll
            for (int q = 0; q < AT_ONCE; ++q)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (!(y[q][k] < tf)) {
                        const unsigned o = key_of(fmaxf(y[q][k], -INFINITY));
                        if (o >= t && e[q] + k < e_hi) {
                            const int to = atomicAdd(&listed, 1);
                            if (to < CAP) list[to] = ((unsigned long long)o << 32) | (unsigned)(0xffffffffu - (unsigned)(e[q] + k));
                        }
                    }
        }
    }

    double total = 0.0;
    {
        const float to = whole_ref(m);                     // (the threads' largest ref, where that is taken)
        double ws = sum * (double)two_to(ref - to);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ws += __shfl_xor_sync(0xffffffffu, ws, o);
        if (lane == 0) wsum[warp] = ws;
    }
    if (__syncthreads_or(sum != sum) || by_difference(m)) {
        // something is no number, or infinite, or very large: once more, in 64 bits from element to element
        double s = 0.0;
        if (m > -INFINITY)
            for (int e = e_lo + tid; e < e_hi; e += ST) {
                const float v = fmaxf(row[e], -INFINITY);
                s += (double)(m == INFINITY ? (v == INFINITY ? 1.f : 0.f)   // the weight lies on the infinite ones alone
                                            : ex2(by_difference(m) ? (v - m) * L : fmaf(v, L, -whole_ref(m))));
            }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        __syncthreads();
        if (lane == 0) wsum[warp] = s;
        __syncthreads();
    }
    if (tid == 0)
#pragma unroll
        for (int w = 0; w < W; ++w) total += wsum[w];

    int n = listed;
    if (n > CAP) {
        // too many reach t (equals, most of them): the value of the last one that belongs, then the index up to which its equals do
        unsigned lo = t, hi = key_m;                       // count(>= lo) >= picks, count(> hi) = 0
        unsigned probe = lo + 1;                           // (most often the many are equal: asked first)
        auto count_of = [&](auto belongs) -> int {
            int mine = 0;
            for (int e = e_lo + tid; e < e_hi; e += ST) mine += belongs(key_of(fmaxf(row[e], -INFINITY)), e);
            return block_count(mine, &cell);
        };
        while (lo < hi) {
            if (count_of([&](unsigned o, int) { return o >= probe; }) >= picks) lo = probe;
            else hi = probe - 1;
            probe = lo + (hi - lo + 1) / 2;
        }
        const int equals = picks - count_of([&](unsigned o, int) { return o > lo; });         // at least 1: the lowest indices
        int b_lo = e_lo, b_hi = e_hi;                      // smallest b with `equals` of them below it
        while (b_lo < b_hi) {
            const int b = b_lo + (b_hi - b_lo) / 2;
            if (count_of([&](unsigned o, int e) { return o == lo && e < b; }) >= equals) b_hi = b;
            else b_lo = b + 1;
        }
        __syncthreads();
        if (tid == 0) listed = 0;
        __syncthreads();
        for (int e = e_lo + tid; e < e_hi; e += ST) {
            const unsigned o = key_of(fmaxf(row[e], -INFINITY));
            if (o > lo || (o == lo && e < b_lo)) {
                const int at = atomicAdd(&listed, 1);
                if (at < CAP) list[at] = ((unsigned long long)o << 32) | (unsigned)(0xffffffffu - (unsigned)e);
            }
        }
        __syncthreads();
        n = min(listed, CAP);
    }
    if (tid == 0) *mine_stat = SliceStat{total, m, n <= 2 * picks ? n : picks};
    if (n <= 2 * picks) {
        for (int i = tid; i < n; i += ST) mine_best[i] = list[i];
        continue;
    }
    for (int i = warp; i < n; i += W) {
        const unsigned long long key = list[i];
        int rank = 0;
        for (int j = lane; j < n; j += 32) rank += list[j] > key;
        rank = __reduce_add_sync(0xffffffffu, rank);
        if (lane == 0 && rank < picks) mine_best[rank] = key;
    }
    }
}

// One CTA a group.  Of the pool's 2 * picks places a slice, the slice's first n are filled.
__global__ void __launch_bounds__(MT)
beam_merge_kernel(const unsigned long long* best, const SliceStat* stat, const float* scores,
                  int vocab, int beams, int slices, int picks, float* out_scores, int* out_rows,
                  int* out_tokens) {
    extern __shared__ unsigned long long pool[];           // [lists][room, as a power of two], where they fit; 0: no element.  Their rounded scores behind
    __shared__ double base[MAX_BEAMS], so_far[MAX_BEAMS];  // log of the row's sum; its score
    __shared__ float row_top[MAX_BEAMS];
    __shared__ double l_score[CAP];
    __shared__ long long l_at[CAP];                        // row of the group << 32 | token
    __shared__ SliceStat held[LISTS];
    __shared__ unsigned wmax[MT / 32], wmin[MT / 32];
    __shared__ unsigned long long best_of[MT / 32];
    __shared__ int cell, listed;
    const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) listed = 0;
    pdl_wait();
    const int lists = beams * slices, room = 2 * picks;
    const unsigned long long* keys = best + (size_t)g * lists * room;
    const SliceStat* of = stat + (size_t)g * lists;
    for (int l = tid; l < min(lists, LISTS); l += MT) held[l] = of[l];
    __syncthreads();
    auto stat_of = [&](int l) -> SliceStat { return l < LISTS ? held[l] : of[l]; };
    // A pool that fits is read once, all of it on its way while the sums are made; its lists lie 1 << places apart.  (1 x 4 beams of 128,256 words
    // 12.4 -> 8.8 us, 32 x 16 with 48 picks 69 -> 66.5: loads that wait for the sums, and a second read of what is taken)
    const int places = 32 - __clz(room - 1);
    const bool fits = lists <= PLACES >> places;
    const int all = fits ? lists << places : 0;
    if (fits) {
        const unsigned to = (unsigned)__cvta_generic_to_shared(pool);
#pragma unroll 4
        for (int at = tid; at < all; at += MT) {
            const int l = at >> places, k = at & ((1 << places) - 1);
            const bool there = k < stat_of(l).n;
            copy_async8(to + 8 * at, there ? keys + (size_t)l * room + k : keys, there);
        }
    }
    for (int b = warp; b < beams; b += MT / 32) {
        const float before = scores[(size_t)g * beams + b];
        float m = -INFINITY;
        for (int i = lane; i < slices; i += 32) m = fmaxf(m, stat_of(b * slices + i).m);
        m = warp_max(m);
        const float ref = whole_ref(m);
        double sum = 0.0;
        for (int i = lane; i < slices; i += 32) {
            const SliceStat s = stat_of(b * slices + i);
            if (s.m == -INFINITY) continue;
            if (!by_difference(m)) {
                if (!by_difference(s.m)) sum += s.sum * two_to(whole_ref(s.m) - ref);        // (else far below: nothing)
            } else if (by_difference(s.m)) {
                sum += s.m == m ? s.sum : s.sum * exp((double)s.m - (double)m);
            } else {
                // (that L is not log2 e to the last bit is made up for by the slice's largest logit: of 65,536 it is 9e-4 of the weight)
                sum += s.sum * exp(0.6931471805599453 * whole_ref(s.m) + (double)s.m * (1.0 - 0.6931471805599453 * (double)L) - (double)m);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            // the largest weight as it is, not to the 2 ulp of its exponential: a token that is all but certain costs nothing
            if (!by_difference(m)) sum += exp2((double)m * (double)L - (double)ref) - (double)ex2(fmaf(m, L, -ref));
            // log of the row's sum; that L is not log2 e to the last bit acts as a factor of the logits, here of the largest
            const double l = log(sum);
            row_top[b] = m;
            so_far[b] = (double)before;
            base[b] = m == INFINITY      ? l
                      : by_difference(m) ? (double)m + l
                                         : l + 0.6931471805599453 * ref + (double)m * (1.0 - 0.6931471805599453 * (double)L);
        }
    }
    __syncthreads();
    // every element of a pool that does not fit, or more than once: a warp four lists, whose loads are in flight together
    auto each = [&](auto use) {
        constexpr int AT_ONCE = 4;
        for (int l0 = warp; l0 < lists; l0 += AT_ONCE * (MT / 32)) {
            int n[AT_ONCE], most = 0;
#pragma unroll
            for (int q = 0; q < AT_ONCE; ++q) {
                const int l = l0 + q * (MT / 32);
                n[q] = l < lists ? stat_of(l).n : 0;
                most = max(most, n[q]);
            }
            for (int k = lane; k < most; k += 32) {
                unsigned long long key[AT_ONCE];
#pragma unroll
                for (int q = 0; q < AT_ONCE; ++q) key[q] = k < n[q] ? keys[(size_t)(l0 + q * (MT / 32)) * room + k] : 0ull;
#pragma unroll
                for (int q = 0; q < AT_ONCE; ++q)
                    if (key[q]) use((l0 + q * (MT / 32)) / slices, key[q]);
            }
        }
    };
    // the element's score; -inf for what is no number (a row all of whose logits are -inf)
    auto score_of = [&](int b, unsigned long long key) -> double {
        const float x = from_ordered((unsigned)(key >> 32));
        double v = so_far[b] + ((double)x - base[b]);
        if (row_top[b] == INFINITY) v = x == INFINITY ? so_far[b] - base[b] : -INFINITY;
        return v == v ? v : -INFINITY;
    };
    auto flat_of = [&](int b, unsigned long long key) -> long long {
        return (long long)b * vocab + (long long)(0xffffffffu - (unsigned)(key & 0xffffffffu));
    };
    asm volatile("cp.async.wait_all;\n" ::: "memory");     // (a thread reads what it has fetched itself)
    // 32-bit keys for the search: rounding keeps the order, and equals after rounding are all gathered
    unsigned mine = 0;
    // (l + 1/2) / slices rounds down to l's row: l is below 2^13, so it is off by 2^-9 of 1 / slices at most, and half of that away from a whole number
    const float a_row = 1.f / (float)slices;
    auto row_of = [&](int at) -> int { return (int)(((float)(at >> places) + 0.5f) * a_row); };
    unsigned* const rounded = reinterpret_cast<unsigned*>(pool + all);
    if (fits) {
#pragma unroll 4
        for (int at = tid; at < all; at += MT) {
            const unsigned long long key = pool[at];
            const unsigned o = key ? ordered((float)score_of(row_of(at), key)) : 0u;
            rounded[at] = o;
            mine = max(mine, o);
        }
    } else {
        each([&](int b, unsigned long long key) { mine = max(mine, ordered((float)score_of(b, key))); });
    }
    unsigned top = __reduce_max_sync(0xffffffffu, mine);
    const unsigned low = __reduce_min_sync(0xffffffffu, mine ? mine : 0xffffffffu);
    if (lane == 0) { wmax[warp] = top; wmin[warp] = low; }
    const int holders = __syncthreads_count(mine != 0);
    top = __reduce_max_sync(0xffffffffu, wmax[lane & (MT / 32 - 1)]);
    unsigned t = holders >= picks ? __reduce_min_sync(0xffffffffu, wmin[lane & (MT / 32 - 1)]) : 1;
    if (lists > 1) t = reach(mine, t, top, picks);
    auto take = [&](int b, unsigned long long key) {
        const int at = atomicAdd(&listed, 1);
        if (at < CAP) { l_score[at] = score_of(b, key); l_at[at] = (long long)b << 32 | (0xffffffffu - (unsigned)(key & 0xffffffffu)); }
    };
    if (fits) {
#pragma unroll 4
        for (int at = tid; at < all; at += MT)
            if (rounded[at] >= t) take(row_of(at), pool[at]);                                  // (t is 1 at least)
    } else {
        each([&](int b, unsigned long long key) {
            if (ordered((float)score_of(b, key)) >= t) take(b, key);
        });
    }
    __syncthreads();
    int n = listed;
    if (n > CAP) {
        // too many: the last score that belongs, by bisection over its 64 bits, then the index of its last equal
        auto ordered64 = [](double v) -> unsigned long long {
            const unsigned long long u = (unsigned long long)__double_as_longlong(v);
            return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
        };
        auto count_of = [&](auto belongs) -> int {
            int c = 0;
            each([&](int b, unsigned long long key) { c += belongs(ordered64(score_of(b, key) + 0.0), flat_of(b, key)); });
            return block_count(c, &cell);
        };
        // asked first: whether it is -inf (most words forbidden), or all are equals of the best (the next of two probes)
        unsigned long long lo = ordered64(-INFINITY), hi = ~0ull, probe = lo + 1;
        bool best_next = true;
        while (lo < hi) {
            if (count_of([&](unsigned long long o, long long) { return o >= probe; }) >= picks) lo = probe;
            else hi = probe - 1;
            probe = lo + (hi - lo) / 2 + 1;
            if (best_next && lo < hi) {
                unsigned long long most = 0;
                each([&](int b, unsigned long long key) { most = max(most, ordered64(score_of(b, key) + 0.0)); });
                const unsigned high = __reduce_max_sync(0xffffffffu, (unsigned)(most >> 32));
                const unsigned low = __reduce_max_sync(0xffffffffu, (unsigned)(most >> 32) == high ? (unsigned)most : 0u);
                __syncthreads();
                if (lane == 0) best_of[warp] = (unsigned long long)high << 32 | low;
                __syncthreads();
                for (int w = 0; w < MT / 32; ++w) most = max(most, best_of[w]);
                hi = probe = most;
            }
            best_next = false;
        }
        const int equals = picks - count_of([&](unsigned long long o, long long) { return o > lo; });
        long long f_lo = 0, f_hi = (long long)beams * vocab;
        while (f_lo < f_hi) {
            const long long f = f_lo + (f_hi - f_lo) / 2;
            if (count_of([&](unsigned long long o, long long at) { return o == lo && at < f; }) >= equals) f_hi = f;
            else f_lo = f + 1;
        }
        __syncthreads();
        if (tid == 0) listed = 0;
        __syncthreads();
        each([&](int b, unsigned long long key) {
            const double s = score_of(b, key);
            const unsigned long long o = ordered64(s + 0.0);
            const long long f = flat_of(b, key);
            if (o > lo || (o == lo && f < f_lo)) take(b, key);
        });
        __syncthreads();
        n = min(listed, CAP);
    }
    for (int i = warp; i < n; i += MT / 32) {
        const double s = l_score[i];
        const long long f = l_at[i];
        int rank = 0;
        for (int j = lane; j < n; j += 32) rank += l_score[j] > s || (l_score[j] == s && l_at[j] < f);
        rank = __reduce_add_sync(0xffffffffu, rank);
        if (lane == 0 && rank < picks) {
            const size_t at = (size_t)g * picks + rank;
            out_scores[at] = (float)s;
            out_rows[at] = g * beams + (int)(f >> 32);
            out_tokens[at] = (int)(f & 0xffffffff);
        }
    }
}

int vectors_of(int vocab) { return (vocab + 3) / 4; }

// Slices a row, by about how many us they take: a chunk 0.65 on its way to a CTA, 0.4 of an SM's bandwidth; a slice's end 2, and 1 more for every
// CTA of the SM, since they come to it together.  (us for 2 / 3 / 4 slices: 512 rows of 128,256 64.0 / 65.9 / 67.2, 128 rows 25.5 / 27.6 / 29.1, 128
// rows of 50,021 16.9 / 17.4 / 18.3; 4 rows of 128,256 for 8 / 16 / 32 slices 9.5 / 8.9 / 8.8)
int slices_of(int rows, int vocab, int sms) {
    const int n = vectors_of(vocab), chunks = (n + NV * ST - 1) / (NV * ST);
    int best = chunks;
    double best_cost = -1.;
    for (int s = (chunks + MAX_CHUNKS - 1) / MAX_CHUNKS; s <= chunks; s = s < 64 ? s + 1 : 2 * s) {
        const int a_slice = (n + s - 1) / s, of_slice = (a_slice + NV * ST - 1) / (NV * ST);
        const double an_sm = (double)rows * s / sms, rounds = an_sm > CTAS ? an_sm / CTAS : 1.;
        const double way = 0.65 * of_slice * rounds, stream = 0.4 * of_slice * an_sm;
        const double cost = (way > stream ? way : stream) + rounds * (2. + (an_sm < CTAS ? an_sm : CTAS));
        if (of_slice <= MAX_CHUNKS && (best_cost < 0. || cost < best_cost)) { best = s; best_cost = cost; }
    }
    return best;
}
}  // namespace

// bytes of scratch: a slice's sum and its best
RI_API int ri_beam_select_slices(int rows, int vocab, int sms) { return slices_of(rows, vocab, sms); }

RI_API int ri_beam_select(const float* logits, long long ld, int vocab, const float* scores, int groups, int beams, int picks, int sms,
                          void* scratch, float* out_scores, int* out_rows, int* out_tokens, void* stream) {
    if (groups <= 0) return 0;
    if (beams < 1 || beams > MAX_BEAMS || picks < 1 || picks > MAX_PICKS || vocab < 1 || vocab > (1 << 30) ||
        (long long)beams * vocab < picks || (long long)groups * beams > 65535)
        return (int)cudaErrorInvalidValue;
    const int rows = groups * beams, slices = slices_of(rows, vocab, sms);
    const int a_slice = (vectors_of(vocab) + slices - 1) / slices;
    if ((long long)rows * slices * picks > (1ll << 30)) return (int)cudaErrorInvalidValue;
    SliceStat* stat = (SliceStat*)scratch;
    unsigned long long* best = (unsigned long long*)(stat + (size_t)rows * slices);
    cudaStream_t s = (cudaStream_t)stream;
    constexpr int ring = STAGES * NV * (ST / 32) * 33 * 16;
    static unsigned long long configured = 0;              // devices, a bit each (one that is set twice is set to the same)
    int device = 0;
    RI_CHECKED((int)cudaGetDevice(&device));
    if (device > 63 || !(configured >> device & 1)) {
        RI_CHECKED((int)cudaFuncSetAttribute(beam_slices_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, ring));
        RI_CHECKED((int)cudaFuncSetAttribute(beam_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PLACES * 12));
        if (device <= 63) configured |= 1ull << device;
    }
    RI_CHECKED(ri_launch(beam_slices_kernel, dim3(min(rows * slices, CTAS * sms)), dim3(ST), ring, s, logits, ld, vocab, scores, picks, rows * slices,
                         slices, a_slice, best, stat));
    const int lists = beams * slices, places = 32 - __builtin_clz(2 * picks - 1), pool = lists <= PLACES >> places ? (lists << places) * 12 : 0;
    RI_CHECKED(ri_launch(beam_merge_kernel, dim3(groups), dim3(MT), pool, s, best, stat, scores, vocab, beams, slices, picks, out_scores, out_rows,
                         out_tokens));
    return ri_launch_status();
}

RI_API void ri_set_pdl(int on) { ri_pdl_flag() = on ? 1 : 0; }
