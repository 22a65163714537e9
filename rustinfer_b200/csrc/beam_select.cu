// Beam search's choice: of every group of `beams` rows the `picks` best continuations by
//
//     score(b, t) = scores[b] + x[b, t] - log sum_t' exp x[b, t']
//
// in descending order, equal scores by ascending (row, token).  RustInfer chooses one token a request
// (crates/infer-worker/src/application/sampler_stack.rs:242-351) and has no counterpart.
//
// Within a row a score falls with its logit, so the row's own best `picks` logits are all that can be chosen, and the
// logits are read once: a CTA holds a slice of a row in registers, sums exp(x - slice maximum), and finds the slice's
// best.  These two are all that leaves the CTA; a second kernel, a CTA a group, puts the slices' sums together in 64
// bits, scores what the slices sent in 64 bits and orders it.
//
// The best `picks` of a slice without a sort: let t be a value that at least `picks` threads' own maxima reach; then at
// least `picks` elements reach it and nothing below it is among the best.  t is found by bisection on the maxima, a
// barrier with a count a step, and stops as soon as no more than twice `picks` threads are left.  The few elements that
// reach t are gathered and a warp counts the ones ahead of each: its rank is its place.  A slice in which more than the
// gathering's room reach t (thousands of equal logits, words that are forbidden) finds the last element that belongs
// to the best exactly, by bisection over values and then over indices.
//
// Scores and the sums over slices are 64-bit: the rows of a group compete through the sums, and a choice hangs on
// differences however small.  Weights are 32-bit exponentials, summed in 32 bits over a warp's elements and in 64 from there.
#include "common.cuh"

namespace {
constexpr int ST = 512;                                    // threads of a slice
constexpr int MT = 512;                                    // threads of a group
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

struct SliceStat {                                         // sum of exp(x - m) over a slice
    double sum;
    float m;
    int pad;
};

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
            if (n <= 2 * picks) break;
        } else {
            hi = mid - 1;
        }
    }
    return lo;
}

template <int NV>
__global__ void __launch_bounds__(ST, 2)
beam_slices_kernel(const float* __restrict__ logits, long long ld, int vocab, const float* __restrict__ scores, int picks,
                   int vectors_a_slice, unsigned long long* __restrict__ best, SliceStat* __restrict__ stat) {
    __shared__ unsigned long long list[CAP];
    __shared__ float wmax[ST / 32];
    __shared__ float wsum[ST / 32];
    __shared__ int cell, listed;
    const int slice = blockIdx.x, slices = gridDim.x, r = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned long long* const mine_best = best + ((size_t)r * slices + slice) * picks;
    SliceStat* const mine_stat = stat + (size_t)r * slices + slice;
    if (tid == 0) listed = 0;
    pdl_wait();
    pdl_trigger();
    const float* const row = logits + (size_t)r * ld;
    // An element's thread goes by its index alone, whatever the row's alignment: equal rows get equal sums, and their
    // continuations are equals that go by index.  A row off a 16-byte boundary is read in single elements.
    const bool aligned = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
    const int v0 = slice * vectors_a_slice, v1 = min(v0 + vectors_a_slice, (vocab + 3) >> 2);
    const int e_lo = 4 * v0, e_hi = min(vocab, 4 * v1);    // the slice's elements
    const float s_row = scores[r];
    if (!(s_row > -INFINITY)) {                            // a row without a future: every score -inf, by index
        for (int i = tid; i < picks; i += ST)
            mine_best[i] = e_lo + i < e_hi ? (0x007fffffull << 32) | (unsigned)(0xffffffffu - (unsigned)(e_lo + i)) : 0ull;
        if (tid == 0) *mine_stat = SliceStat{0.0, -INFINITY, 0};
        return;
    }
    float x[4 * NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int v = v0 + i * ST + tid, e = 4 * v;
        if (aligned && v < v1 && e + 4 <= vocab) {
            const float4 f = __ldcs(reinterpret_cast<const float4*>(row + e));
            x[4 * i] = f.x; x[4 * i + 1] = f.y; x[4 * i + 2] = f.z; x[4 * i + 3] = f.w;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) x[4 * i + k] = v < v1 && e + k < vocab ? row[e + k] : -INFINITY;
        }
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4 * NV; ++i) {
        x[i] = fmaxf(x[i], -INFINITY);                     // what is no number has no chance
        top = fmaxf(top, x[i]);
    }
    const unsigned own_top = key_of(top);
    top = from_ordered(__reduce_max_sync(0xffffffffu, own_top));
    if (lane == 0) wmax[warp] = top;
    __syncthreads();
    float m = wmax[lane & (ST / 32 - 1)];
    m = from_ordered(__reduce_max_sync(0xffffffffu, ordered(m)));
    float sum = 0.f;
    if (m == INFINITY) {                                   // the weight lies on the infinite ones alone
#pragma unroll
        for (int i = 0; i < 4 * NV; ++i) sum += x[i] == INFINITY ? 1.f : 0.f;
    } else if (m > -INFINITY) {
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) part[k] += exp2f((x[4 * i + k] - m) * 1.4426950408889634f);
        sum = (part[0] + part[1]) + (part[2] + part[3]);
    }
    sum = warp_sum(sum);
    if (lane == 0) wsum[warp] = sum;

    // a value that the slice's best all reach
    const int count = e_hi - e_lo;
    unsigned t = 0;
    if (count > 2 * picks) t = reach(own_top, 0x007fffffu, ordered(m), picks);
    if (own_top >= t) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = 4 * (v0 + i * ST + tid);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const unsigned o = key_of(x[4 * i + k]);
                if (o >= t && e + k < e_hi) {
                    const int at = atomicAdd(&listed, 1);
                    if (at < CAP) list[at] = ((unsigned long long)o << 32) | (unsigned)(0xffffffffu - (unsigned)(e + k));
                }
            }
        }
    }
    __syncthreads();
    if (tid == 0) {
        double total = 0.0;
        for (int w = 0; w < ST / 32; ++w) total += (double)wsum[w];
        *mine_stat = SliceStat{total, m, 0};
    }
    int n = listed;
    if (n > CAP) {
        // too many reach t: the value of the last one that belongs, then the index up to which its equals do
        unsigned lo = t, hi = ordered(m);                  // count(>= lo) >= picks, count(> hi) = 0
        unsigned probe = lo + 1;                           // (most often the many are equal: asked first)
        while (lo < hi) {
            int c = 0;
#pragma unroll
            for (int i = 0; i < 4 * NV; ++i) {
                const int e = 4 * (v0 + (i >> 2) * ST + tid) + (i & 3);
                c += key_of(x[i]) >= probe && e < e_hi;
            }
            if (block_count(c, &cell) >= picks) lo = probe;
            else hi = probe - 1;
            probe = lo + (hi - lo + 1) / 2;
        }
        int c = 0;
#pragma unroll
        for (int i = 0; i < 4 * NV; ++i) {
            const int e = 4 * (v0 + (i >> 2) * ST + tid) + (i & 3);
            c += key_of(x[i]) > lo && e < e_hi;
        }
        const int equals = picks - block_count(c, &cell);   // at least 1 of those with the value itself, the lowest indices
        int b_lo = e_lo, b_hi = e_hi;                       // smallest b with `equals` of them below it
        while (b_lo < b_hi) {
            const int b = b_lo + (b_hi - b_lo) / 2;
            c = 0;
#pragma unroll
            for (int i = 0; i < 4 * NV; ++i) {
                const int e = 4 * (v0 + (i >> 2) * ST + tid) + (i & 3);
                c += key_of(x[i]) == lo && e < b;
            }
            if (block_count(c, &cell) >= equals) b_hi = b;
            else b_lo = b + 1;
        }
        __syncthreads();
        if (tid == 0) listed = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4 * NV; ++i) {
            const int e = 4 * (v0 + (i >> 2) * ST + tid) + (i & 3);
            const unsigned o = key_of(x[i]);
            if (o > lo ? e < e_hi : o == lo && e < b_lo) {
                const int at = atomicAdd(&listed, 1);
                if (at < CAP) list[at] = ((unsigned long long)o << 32) | (unsigned)(0xffffffffu - (unsigned)e);
            }
        }
        __syncthreads();
        n = min(listed, CAP);
    }
    for (int i = n + tid; i < picks; i += ST) mine_best[i] = 0ull;          // fewer elements than picks
    for (int i = warp; i < n; i += ST / 32) {
        const unsigned long long key = list[i];
        int rank = 0;
        for (int j = lane; j < n; j += 32) rank += list[j] > key;
        rank = __reduce_add_sync(0xffffffffu, rank);
        if (lane == 0 && rank < picks) mine_best[rank] = key;
    }
}

// One CTA a group.  An element of the pool is a row's, a slice's and a rank's; 0 where a slice had fewer.
__global__ void __launch_bounds__(MT)
beam_merge_kernel(const unsigned long long* __restrict__ best, const SliceStat* __restrict__ stat, const float* __restrict__ scores,
                  int vocab, int beams, int slices, int picks, float* __restrict__ out_scores, int* __restrict__ out_rows,
                  int* __restrict__ out_tokens) {
    __shared__ double base[MAX_BEAMS];                     // scores[b] - log of the row's sum
    __shared__ float row_top[MAX_BEAMS];
    __shared__ double l_score[CAP];
    __shared__ long long l_flat[CAP];
    __shared__ unsigned wmax[MT / 32];
    __shared__ int cell, listed;
    const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) listed = 0;
    pdl_wait();
    for (int b = warp; b < beams; b += MT / 32) {
        const SliceStat* s = stat + ((size_t)g * beams + b) * slices;
        float m = -INFINITY;
        for (int i = lane; i < slices; i += 32) m = fmaxf(m, s[i].m);
        m = warp_max(m);
        double sum = 0.0;
        for (int i = lane; i < slices; i += 32)
            if (s[i].m > -INFINITY) sum += s[i].m == m ? s[i].sum : s[i].sum * exp((double)s[i].m - (double)m);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            row_top[b] = m;
            base[b] = m == INFINITY ? (double)scores[(size_t)g * beams + b] - log(sum) : (double)m + log(sum);
        }
    }
    __syncthreads();
    // rank by rank, so that neighbouring threads hold the heads of the lists
    const int lists = beams * slices, pool = lists * picks;
    const unsigned long long* keys = best + (size_t)g * pool;
    auto key_at = [&](int i, int& b) -> unsigned long long {
        const int rank = i / lists, list = i - rank * lists;
        b = list / slices;
        return keys[(size_t)list * picks + rank];
    };
    // the element's score; -inf for what is no number (a row all of whose logits are -inf)
    auto score_of = [&](int b, unsigned long long key) -> double {
        const float x = from_ordered((unsigned)(key >> 32)), m = row_top[b];
        double v;
        if (m == INFINITY) v = x == INFINITY ? base[b] : -INFINITY;
        else v = x == -INFINITY ? -INFINITY : (double)scores[(size_t)g * beams + b] + ((double)x - base[b]);
        return v == v ? v : -INFINITY;
    };
    auto flat_of = [&](int b, unsigned long long key) -> long long {
        return (long long)b * vocab + (long long)(0xffffffffu - (unsigned)(key & 0xffffffffu));
    };
    // 32-bit keys for the search: rounding keeps the order, and equals after rounding are all gathered
    unsigned mine = 0;
    for (int i = tid; i < pool; i += MT) {
        int b;
        const unsigned long long key = key_at(i, b);
        if (key) mine = max(mine, ordered((float)score_of(b, key)));
    }
    unsigned top = __reduce_max_sync(0xffffffffu, mine);
    if (lane == 0) wmax[warp] = top;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, wmax[lane & (MT / 32 - 1)]);
    unsigned t = 1;
    if (pool > 2 * picks) t = reach(mine, 1, top, picks);
    for (int i = tid; i < pool; i += MT) {
        int b;
        const unsigned long long key = key_at(i, b);
        if (!key) continue;
        const double s = score_of(b, key);
        if (ordered((float)s) >= t) {
            const int at = atomicAdd(&listed, 1);
            if (at < CAP) { l_score[at] = s; l_flat[at] = flat_of(b, key); }
        }
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
            for (int i = tid; i < pool; i += MT) {
                int b;
                const unsigned long long key = key_at(i, b);
                if (key) c += belongs(ordered64(score_of(b, key) + 0.0), flat_of(b, key));
            }
            return block_count(c, &cell);
        };
        unsigned long long lo = 0, hi = ~0ull;
        while (lo < hi) {
            const unsigned long long mid = lo + (hi - lo) / 2 + 1;
            if (count_of([&](unsigned long long o, long long) { return o >= mid; }) >= picks) lo = mid;
            else hi = mid - 1;
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
        for (int i = tid; i < pool; i += MT) {
            int b;
            const unsigned long long key = key_at(i, b);
            if (!key) continue;
            const double s = score_of(b, key);
            const unsigned long long o = ordered64(s + 0.0);
            const long long f = flat_of(b, key);
            if (o > lo || (o == lo && f < f_lo)) {
                const int at = atomicAdd(&listed, 1);
                if (at < CAP) { l_score[at] = s; l_flat[at] = f; }
            }
        }
        __syncthreads();
        n = min(listed, CAP);
    }
    for (int i = warp; i < n; i += MT / 32) {
        const double s = l_score[i];
        const long long f = l_flat[i];
        int rank = 0;
        for (int j = lane; j < n; j += 32) rank += l_score[j] > s || (l_score[j] == s && l_flat[j] < f);
        rank = __reduce_add_sync(0xffffffffu, rank);
        if (lane == 0 && rank < picks) {
            const size_t at = (size_t)g * picks + rank;
            out_scores[at] = (float)s;
            out_rows[at] = g * beams + (int)(f / vocab);
            out_tokens[at] = (int)(f % vocab);
        }
    }
}

int vectors_of(int vocab) { return (vocab + 3) / 4; }

// 16-byte loads a thread: as many as leave two CTAs an SM something to do.  Few rows go in more and smaller slices
int vectors_a_thread(int rows, int vocab, int sms) {
    const int n = vectors_of(vocab);
    for (int nv = 8; nv > 2; nv >>= 1)
        if ((long long)rows * ((n + nv * ST - 1) / (nv * ST)) >= 2ll * sms) return nv;
    return 2;
}
int slices_of(int rows, int vocab, int sms) {
    const int a_slice = vectors_a_thread(rows, vocab, sms) * ST;
    return (vectors_of(vocab) + a_slice - 1) / a_slice;
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
    const int rows = groups * beams, nv = vectors_a_thread(rows, vocab, sms), slices = slices_of(rows, vocab, sms);
    const int a_slice = (vectors_of(vocab) + slices - 1) / slices;
    SliceStat* stat = (SliceStat*)scratch;
    unsigned long long* best = (unsigned long long*)(stat + (size_t)rows * slices);
    const dim3 grid(slices, rows);
    cudaStream_t s = (cudaStream_t)stream;
    auto kernel = nv == 8 ? beam_slices_kernel<8> : nv == 4 ? beam_slices_kernel<4> : beam_slices_kernel<2>;
    RI_CHECKED(ri_launch(kernel, grid, dim3(ST), 0, s, logits, ld, vocab, scores, picks, a_slice, best, stat));
    RI_CHECKED(ri_launch(beam_merge_kernel, dim3(groups), dim3(MT), 0, s, best, stat, scores, vocab, beams, slices, picks, out_scores, out_rows,
                         out_tokens));
    return ri_launch_status();
}

RI_API void ri_set_pdl(int on) { ri_pdl_flag() = on ? 1 : 0; }
