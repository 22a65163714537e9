// What a request's beams leave behind and take over: rows of a cache moved inside the device.
//
//   reorder_rows  rows[r] <- rows[parents[r]] within every group of beams, in place, in every layer
//   copy_pages    page dst[i] <- page src[i], in every layer
//
// A row is a request's state slot, or the page its next token goes to; of a page only the tokens in use are moved.  RustInfer keeps
// one sequence a request and copies nothing (crates/infer-worker/src/domain/global_kv_alloc.rs:129-194).
//
// Both are streams: a byte is read once and written once.  In place without a second buffer: a thread owns one column of 16 bytes
// and moves it through all rows of its group, so no two threads meet, and it makes the moves in an order in which no row is
// overwritten before its last reader has read it.  After a step of beam search every source is a row that stays (a beam that
// has a continuation keeps its row), so any order will do and the loads of several moves are in flight together; a mapping in which
// a source moves too is put in order first, and a cycle goes through one register.
#include "common.cuh"

namespace {
constexpr int RT = 256;                                    // threads
constexpr int MAX_BEAMS = 64;
constexpr int TEMP = -1;                                   // in place of a row: the thread's register

// How far into a row a move reaches: rows are `segments` runs of `seg` vectors, of which the first tokens * a_token are in use
struct Extent {
    int seg;                                               // vectors a segment
    int a_token;                                           // vectors a token takes in it
    const int* tokens;                                     // by row of the call; null: whole rows
};
__device__ __forceinline__ int used_of(const Extent& x, int i) {
    if (!x.tokens) return x.seg;
    return (int)min((long long)x.seg, max(0ll, (long long)x.tokens[i] * x.a_token));
}

template <typename V, int U>
__global__ void __launch_bounds__(RT)
reorder_rows_kernel(V* store, long long total, int row_vectors, const int* rows, const int* parents,
                    int beams, Extent extent) {
    __shared__ int m_src[2 * MAX_BEAMS], m_dst[2 * MAX_BEAMS], m_used[2 * MAX_BEAMS];
    __shared__ int n_moves, cyclic;
    pdl_wait();
    const int g0 = blockIdx.z * beams, tid = threadIdx.x, lane = tid & 31;
    if (tid < 32) {
        // two rows a lane
        int src[2], dst[2], par[2], used[2];
        unsigned long long moving = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = lane + 32 * h;
            src[h] = dst[h] = TEMP; par[h] = r; used[h] = 0;
            bool moves = false;
            if (r < beams) {
                const int p = parents[g0 + r] - g0;        // a row outside the group is no parent: the row stays
                if (p >= 0 && p < beams && p != r) {
                    par[h] = p;
                    dst[h] = rows[g0 + r];
                    src[h] = rows[g0 + p];
                    used[h] = used_of(extent, g0 + r);
                    moves = dst[h] >= 0 && dst[h] < total && src[h] >= 0 && src[h] < total && dst[h] != src[h] && used[h] > 0;
                }
            }
            moving |= (unsigned long long)__ballot_sync(0xffffffffu, moves) << (32 * h);
        }
        auto read_by = [&](unsigned long long of) -> unsigned long long {           // rows that the moves `of` read
            unsigned lo = 0, hi = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if ((of >> (lane + 32 * h) & 1) && par[h] < MAX_BEAMS) (par[h] < 32 ? lo : hi) |= 1u << (par[h] & 31);
            return (unsigned long long)__reduce_or_sync(0xffffffffu, hi) << 32 | __reduce_or_sync(0xffffffffu, lo);
        };
        int n = 0, through = 0;
        unsigned long long pending = moving;
        while (pending) {
            unsigned long long free = pending & ~read_by(pending);                   // nobody waits for what these hold
            if (!free) {
                // cycles alone are left: the lowest row's content into the register, its reader takes it from there
                const int d = __ffsll((long long)pending) - 1;
                const int dr = __shfl_sync(0xffffffffu, d < 32 ? dst[0] : dst[1], d & 31);
                if (lane == 0) { m_src[n] = dr; m_dst[n] = TEMP; m_used[n] = extent.seg; }
                ++n;
                through = 1;
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if ((pending >> (lane + 32 * h) & 1) && par[h] == d) { src[h] = TEMP; par[h] = MAX_BEAMS; }
                free = 1ull << d;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const unsigned long long below = h ? (free & ((1ull << (lane + 32)) - 1)) : (free & ((1ull << lane) - 1));
                if (free >> (lane + 32 * h) & 1) {
                    const int at = n + __popcll(below);
                    m_src[at] = src[h]; m_dst[at] = dst[h]; m_used[at] = used[h];
                }
            }
            n += __popcll(free);
            pending &= ~free;
        }
        if (lane == 0) { n_moves = n; cyclic = through; }
    }
    __syncthreads();
    const int n = n_moves;
    if (n == 0) return;
    V* const layer = store + (size_t)blockIdx.y * total * row_vectors;
    const int c0 = blockIdx.x * (RT * U) + tid;
    if (cyclic) {
        for (int u = 0; u < U; ++u) {
            const int c = c0 + u * RT;
            if (c >= row_vectors) break;
            const int off = c % extent.seg;
            V held = {};
            for (int i = 0; i < n; ++i) {
                if (off >= m_used[i]) continue;
                const V v = m_src[i] == TEMP ? held : layer[(size_t)m_src[i] * row_vectors + c];
                if (m_dst[i] == TEMP) held = v;
                else layer[(size_t)m_dst[i] * row_vectors + c] = v;
            }
        }
        return;
    }
    int off[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int c = c0 + u * RT;
        off[u] = c >= row_vectors ? 0x7fffffff : c % extent.seg;
    }
    constexpr int B = 4;                                   // moves whose loads are in flight together
    for (int i0 = 0; i0 < n; i0 += B) {
        V v[B][U];
#pragma unroll
        for (int i = 0; i < B; ++i)
            if (i0 + i < n) {
                const V* from = layer + (size_t)m_src[i0 + i] * row_vectors + c0;
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (off[u] < m_used[i0 + i]) v[i][u] = from[u * RT];
            }
#pragma unroll
        for (int i = 0; i < B; ++i)
            if (i0 + i < n) {
                V* to = layer + (size_t)m_dst[i0 + i] * row_vectors + c0;
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (off[u] < m_used[i0 + i]) to[u * RT] = v[i][u];
            }
    }
}

template <typename V, int U>
__global__ void __launch_bounds__(RT)
copy_pages_kernel(V* store, long long total, int row_vectors, int chunks, const int* src, const int* dst,
                  Extent extent) {
    pdl_wait();
    const int i = blockIdx.x / chunks, chunk = blockIdx.x - i * chunks;
    const int s = src[i], d = dst[i];
    if (s < 0 || s >= total || d < 0 || d >= total || s == d) return;
    const int used = used_of(extent, i), c0 = chunk * (RT * U) + threadIdx.x;
    V* const layer = store + (size_t)blockIdx.y * total * row_vectors;
    const V* from = layer + (size_t)s * row_vectors + c0;
    V* to = layer + (size_t)d * row_vectors + c0;
    V v[U];
    bool in[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int c = c0 + u * RT;
        in[u] = c < row_vectors && c % extent.seg < used;
        if (in[u]) v[u] = from[u * RT];
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (in[u]) to[u * RT] = v[u];
}

// Vectors of the widest type that the rows', the segments' and the tokens' bytes and the address allow
template <typename F>
int by_vector(const void* store, long long row_bytes, long long seg_bytes, long long token_bytes, F launch) {
    const long long all = (long long)(reinterpret_cast<uintptr_t>(store) | (uintptr_t)row_bytes | (uintptr_t)seg_bytes | (uintptr_t)token_bytes);
    if (all % 16 == 0) return launch(uint4{}, 16);
    if (all % 4 == 0) return launch(unsigned{}, 4);
    if (all % 2 == 0) return launch((unsigned short)0, 2);
    return launch((unsigned char)0, 1);
}
bool sizes_hold(long long total, long long row_bytes, long long seg_bytes, long long token_bytes, int layers) {
    return total > 0 && row_bytes > 0 && row_bytes < (1ll << 31) && seg_bytes > 0 && row_bytes % seg_bytes == 0 && token_bytes > 0 &&
           seg_bytes % token_bytes == 0 && layers <= 65535;
}
}  // namespace

// store: [layers][total rows][row_bytes].  tokens null: whole rows (seg_bytes = token_bytes = row_bytes).
RI_API int ri_reorder_rows(void* store, int layers, long long total, long long row_bytes, long long seg_bytes, long long token_bytes,
                           const int* rows, const int* parents, int groups, int beams, const int* tokens, void* stream) {
    if (groups <= 0 || layers <= 0) return 0;
    if (beams < 1 || beams > MAX_BEAMS || groups > 65535 || !sizes_hold(total, row_bytes, seg_bytes, token_bytes, layers))
        return (int)cudaErrorInvalidValue;
    return by_vector(store, row_bytes, seg_bytes, token_bytes, [&](auto v, int size) -> int {
        using V = decltype(v);
        constexpr int U = 2;
        const int n = (int)(row_bytes / size);
        const Extent x{(int)(seg_bytes / size), (int)(token_bytes / size), tokens};
        RI_CHECKED(ri_launch(reorder_rows_kernel<V, U>, dim3((n + RT * U - 1) / (RT * U), layers, groups), dim3(RT), 0, (cudaStream_t)stream,
                             (V*)store, total, n, rows, parents, beams, x));
        return ri_launch_status();
    });
}

RI_API int ri_copy_pages(void* store, int layers, long long total, long long row_bytes, long long seg_bytes, long long token_bytes, const int* src,
                         const int* dst, int pairs, const int* tokens, void* stream) {
    if (pairs <= 0 || layers <= 0) return 0;
    if (!sizes_hold(total, row_bytes, seg_bytes, token_bytes, layers)) return (int)cudaErrorInvalidValue;
    return by_vector(store, row_bytes, seg_bytes, token_bytes, [&](auto v, int size) -> int {
        using V = decltype(v);
        constexpr int U = 4;
        const int n = (int)(row_bytes / size), chunks = (n + RT * U - 1) / (RT * U);
        if ((long long)pairs * chunks > 0x7fffffffll) return (int)cudaErrorInvalidValue;
        const Extent x{(int)(seg_bytes / size), (int)(token_bytes / size), tokens};
        RI_CHECKED(ri_launch(copy_pages_kernel<V, U>, dim3(pairs * chunks, layers), dim3(RT), 0, (cudaStream_t)stream, (V*)store, total, n,
                             chunks, src, dst, x));
        return ri_launch_status();
    });
}
