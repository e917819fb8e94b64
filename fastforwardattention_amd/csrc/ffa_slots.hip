// Moves of cache slots (gfx950): the accepted path of a drafted tree, and eviction by accumulated
// attention weight.  Also the dispatch of the tree kernels over the element types.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "ffa_cache_ops.h"
#include "ffa_device.h"

namespace ffa {

int launch_tree(int precision, int head_dim, const TreeParams& P, const TreePlan& plan, void* stream) {
    if (precision == FFA_PRECISION_F16) return launch_tree_f16(P, head_dim, plan, stream);
    if (precision == FFA_PRECISION_BF16) return launch_tree_bf16(P, head_dim, plan, stream);
    return launch_tree_f32(P, head_dim, plan, stream);
}

// ---------------------------------------------------------------------------------------
// Commit.  One wave moves the accepted slots of 8 chunk columns (128 bytes a slot) of one pair, K
// or V; path_len <= 64, so all of them are in its registers before the first is stored.  Bound by
// latency: a few KB a pair.
__device__ __forceinline__ void all_loaded() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

template <int NCH>
__global__ void __launch_bounds__(256) ffa_commit_kernel(const CommitParams P) {
    constexpr int NB = NCH % 8 == 0 ? 8 : NCH / 2 <= 8 ? NCH / 2 : NCH / 4;  // chunks of a column block (Dh = 80: 5)
    constexpr int COLS = NCH / NB;
    constexpr int RPI = 64 / NB;  // rows of V an access covers
    const int lane = threadIdx.x & 63;
    const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int pairs = P.B * P.H;
    const int col = (int)(unit % (2 * COLS));
    const long long rest = unit / (2 * COLS);
    const int pair = (int)(rest % pairs), cache = (int)(rest / pairs);
    if (cache >= P.n_caches) return;
    const int b = pair / P.H;
    const int base = P.lengths ? min(max(P.lengths[b], 0), P.t) : P.t;
    const int n = min(max(P.accepted[b], 0), P.path_len);
    if (lane >= n && n == 0) return;
    // Old slot of path entry `lane`, inside the cache whatever the entry holds.
    const int entry = P.path[(size_t)b * P.path_len + min(lane, P.path_len - 1)];
    const int from = base + min(max(entry, 0), P.Lmax - 1 - base);
    const int c0 = (col >> 1) * NB;
    if ((col & 1) == 0) {
        u32x4_t* kc = static_cast<u32x4_t*>(P.k[cache]) + ((size_t)pair * NCH + c0) * P.Lmax;
        const bool move = lane < n && from != base + lane;
        u32x4_t x[NB];
#pragma unroll
        for (int c = 0; c < NB; ++c) x[c] = kc[(size_t)c * P.Lmax + from];
        all_loaded();
        if (move) {
#pragma unroll
            for (int c = 0; c < NB; ++c) kc[(size_t)c * P.Lmax + base + lane] = x[c];
        }
    } else {
        u32x4_t* vc = static_cast<u32x4_t*>(P.v[cache]) + (size_t)pair * P.Lmax * NCH + c0;
        constexpr int IT = (64 + RPI - 1) / RPI;
        u32x4_t x[IT];
        const int r0 = lane / NB, c = lane % NB;
#pragma unroll
        for (int it = 0; it < IT; ++it) {
            const int row = it * RPI + r0;
            const int src = __shfl(from, row & 63);
            x[it] = u32x4_t{0, 0, 0, 0};
            if (r0 < RPI && row < n) x[it] = vc[(size_t)src * NCH + c];
        }
        all_loaded();
#pragma unroll
        for (int it = 0; it < IT; ++it) {
            const int row = it * RPI + r0;
            if (r0 < RPI && row < n) vc[(size_t)(base + row) * NCH + c] = x[it];
        }
    }
}

// ---------------------------------------------------------------------------------------
// Eviction, first kernel: which slots stay.  One workgroup a pair.  Weights become 32-bit keys in
// the order of the ranking, padding 0, NaN 1; a radix select over 8-bit digits finds the smallest
// key that stays and how many of its equals do; then every wave walks its stretch of the slots in
// order and writes the chosen ones behind those of the stretches before it.
constexpr int kSelectThreads = 1024;

__device__ __forceinline__ uint32_t rank_key(float w) {
    if (w != w) return 1;
    const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.f);  // -0 ranks as +0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kSelectThreads) ffa_evict_select_kernel(const EvictParams P) {
    constexpr int NW = kSelectThreads / 64;
    __shared__ unsigned s_hist[256];
    __shared__ unsigned s_wave[NW][2];
    __shared__ unsigned s_digit, s_above;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int pairs = P.B * P.H;
    const int cache = blockIdx.x / pairs, pair = blockIdx.x % pairs, b = pair / P.H;
    const int length = P.lengths ? min(max(P.lengths[b], 0), P.t) : P.t;
    const int first = P.first_keys ? min(max(P.first_keys[b], 0), length) : 0;
    const float* w = P.w_src[cache] + (size_t)pair * P.src_len;
    float* to = P.w_dst[cache] + (size_t)pair * P.dst_len;
    int* kept = P.kept + ((size_t)cache * pairs + pair) * P.keep;
    const int stay = min(length, P.keep);
    const int tail = length - P.recent;  // slots from here on stay (if length > keep, which is >= recent)
    const int budget = P.keep - P.recent;

    if (length <= P.keep) {
        for (int j = tid; j < P.keep; j += kSelectThreads) kept[j] = j < length ? j : -1;
    } else {
        uint32_t prefix = 0, need = budget;  // keys whose upper digits equal prefix's: `need` of them stay
        if (budget > 0) {
            for (int shift = 24; shift >= 0; shift -= 8) {
                if (tid < 256) s_hist[tid] = 0;
                __syncthreads();
                for (int j = tid; j < tail; j += kSelectThreads) {
                    const uint32_t k = j < first ? 0 : rank_key(w[j]);
                    if (shift == 24 || ((k ^ prefix) >> (shift + 8)) == 0) atomicAdd(&s_hist[(k >> shift) & 255], 1u);
                }
                __syncthreads();
                if (wave == 0) {
                    // Counts from the top digit down: lane i holds digits 255 - 4 i .. 252 - 4 i.
                    unsigned n[4], sum = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        n[e] = s_hist[255 - 4 * lane - e];
                        sum += n[e];
                    }
                    unsigned incl = sum;
#pragma unroll
                    for (int d = 1; d < 64; d <<= 1) {
                        const unsigned up = __shfl_up(incl, d);
                        if (lane >= d) incl += up;
                    }
                    unsigned above = incl - sum;
                    if (above < need && incl >= need) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (above < need && above + n[e] >= need) {
                                s_digit = 255 - 4 * lane - e;
                                s_above = above;
                                break;
                            }
                            above += n[e];
                        }
                    }
                }
                __syncthreads();
                prefix |= s_digit << shift;
                need -= s_above;
            }
        }
        // Stretches of whole wave steps, in slot order.
        const int steps = (tail + 64 * NW - 1) / (64 * NW);
        const int lo = wave * steps * 64, hi = min(lo + steps * 64, tail);
        unsigned n_more = 0, n_equal = 0;
        if (budget > 0) {
            for (int j0 = lo; j0 < hi; j0 += 64) {
                const int j = j0 + lane;
                const uint32_t k = j < first ? 0 : j < hi ? rank_key(w[j]) : 0;
                n_more += __popcll(__ballot(j < hi && k > prefix));
                n_equal += __popcll(__ballot(j < hi && k == prefix));
            }
        }
        if (lane == 0) {
            s_wave[wave][0] = n_more;
            s_wave[wave][1] = n_equal;
        }
        __syncthreads();
        unsigned more = 0, equal = 0;
        for (int i = 0; i < wave; ++i) {
            more += s_wave[i][0];
            equal += s_wave[i][1];
        }
        if (budget > 0) {
            const unsigned long long below = (1ull << lane) - 1;
            for (int j0 = lo; j0 < hi; j0 += 64) {
                const int j = j0 + lane;
                const uint32_t k = j < first ? 0 : j < hi ? rank_key(w[j]) : 0;
                const unsigned long long m_more = __ballot(j < hi && k > prefix);
                const unsigned long long m_equal = __ballot(j < hi && k == prefix);
                const unsigned e = equal + __popcll(m_equal & below);
                const bool chosen = (m_more >> lane & 1) || ((m_equal >> lane & 1) && e < need);
                if (chosen) kept[more + __popcll(m_more & below) + min(e, need)] = j;
                more += __popcll(m_more);
                equal += __popcll(m_equal);
            }
        }
        for (int j = tid; j < P.recent; j += kSelectThreads) kept[budget + j] = tail + j;
    }
    __syncthreads();
    // Weights follow.  In place: a chunk's sources lie at or behind its targets, and behind the
    // targets of all chunks before it, so only the loads and stores of one chunk need the barrier.
    for (int j0 = 0; j0 < stay; j0 += kSelectThreads) {
        const int j = j0 + tid;
        float x = 0.f;
        if (j < stay) x = w[kept[j]];
        __syncthreads();
        if (j < stay) to[j] = x;
    }
}

// Eviction, second kernel: the rows of K and V.  One wave takes one chunk row of a pair's K (64
// slots of 16 bytes an access) or one column block of its V (8 chunks x 8 slots an access) through
// all kept slots in order.  In place this needs no other synchronisation: kept[j] >= j, so what is
// stored for slots [j, j + n) can only overwrite sources of entries before j + n, which this wave
// has loaded already, and no other wave touches the column.  Two batches of loads are in flight.
template <int NCH>
__global__ void __launch_bounds__(256) ffa_evict_move_kernel(const EvictParams P) {
    constexpr int NB = NCH % 8 == 0 ? 8 : NCH / 2 <= 8 ? NCH / 2 : NCH / 4;
    constexpr int COLS = NCH / NB;
    constexpr int RPI = 64 / NB;
    constexpr int U = 8;  // accesses of a batch
    const int lane = threadIdx.x & 63;
    const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int pairs = P.B * P.H;
    constexpr int UNITS = NCH + COLS;
    const int col = (int)(unit % UNITS);
    const long long rest = unit / UNITS;
    const int pair = (int)(rest % pairs), cache = (int)(rest / pairs);
    if (cache >= P.n_caches) return;
    const int b = pair / P.H;
    const int length = P.lengths ? min(max(P.lengths[b], 0), P.t) : P.t;
    const int stay = min(length, P.keep);
    const bool is_k = col < NCH;
    const u32x4_t* src;
    u32x4_t* dst;
    int stride, rows, r0;  // chunks between slots, slots of an access, this lane's slot
    if (is_k) {
        src = static_cast<const u32x4_t*>(P.k_src[cache]) + ((size_t)pair * NCH + col) * P.src_len;
        dst = static_cast<u32x4_t*>(P.k_dst[cache]) + ((size_t)pair * NCH + col) * P.dst_len;
        stride = 1; rows = 64; r0 = lane;
    } else {
        const int c0 = (col - NCH) * NB + lane % NB;
        src = static_cast<const u32x4_t*>(P.v_src[cache]) + (size_t)pair * P.src_len * NCH + c0;
        dst = static_cast<u32x4_t*>(P.v_dst[cache]) + (size_t)pair * P.dst_len * NCH + c0;
        stride = NCH; rows = RPI; r0 = lane / NB;
    }
    const bool active = is_k || r0 < RPI;
    const bool in_place = src == dst;
    if (in_place && length <= P.keep) return;
    const int* kept = P.kept + ((size_t)cache * pairs + pair) * P.keep;

    int from[2][U];
    u32x4_t x[2][U];
    auto load = [&](int s, int j0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + u * rows + r0;
            from[s][u] = active && j < stay ? kept[j] : -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (in_place && from[s][u] == j0 + u * rows + r0) from[s][u] = -1;
            x[s][u] = u32x4_t{0, 0, 0, 0};
            if (from[s][u] >= 0) x[s][u] = src[(size_t)from[s][u] * stride];
        }
    };
    auto store = [&](int s, int j0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (from[s][u] >= 0) dst[(size_t)(j0 + u * rows + r0) * stride] = x[s][u];
    };
    const int batch = U * rows;
    load(0, 0);
    for (int j0 = 0; j0 < stay; j0 += 2 * batch) {
        load(1, j0 + batch);
        store(0, j0);
        load(0, j0 + 2 * batch);
        store(1, j0 + batch);
    }
}

// ---------------------------------------------------------------------------------------
static int launched() { return hipGetLastError() == hipSuccess ? FFA_OK : FFA_ERR_LAUNCH; }

template <int NCH> static int commit_nch(const CommitParams& P, hipStream_t st) {
    constexpr int NB = NCH % 8 == 0 ? 8 : NCH / 2 <= 8 ? NCH / 2 : NCH / 4;
    const long long units = (long long)P.n_caches * P.B * P.H * (2 * NCH / NB);
    if (units == 0) return FFA_OK;
    hipLaunchKernelGGL(ffa_commit_kernel<NCH>, dim3((unsigned)((units + 3) / 4)), dim3(256), 0, st, P);
    return launched();
}

int launch_commit(const CommitParams& P, int head_dim, int elem_bytes, void* stream) {
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    switch (head_dim * elem_bytes / 16) {
        case 8: return commit_nch<8>(P, st);
        case 10: return commit_nch<10>(P, st);
        case 16: return commit_nch<16>(P, st);
        case 20: return commit_nch<20>(P, st);
        case 32: return commit_nch<32>(P, st);
        case 64: return commit_nch<64>(P, st);
        default: return FFA_ERR_HEAD_DIM;
    }
}

template <int NCH> static int evict_nch(const EvictParams& P, hipStream_t st) {
    constexpr int NB = NCH % 8 == 0 ? 8 : NCH / 2 <= 8 ? NCH / 2 : NCH / 4;
    const long long lines = (long long)P.n_caches * P.B * P.H;
    hipLaunchKernelGGL(ffa_evict_select_kernel, dim3((unsigned)lines), dim3(kSelectThreads), 0, st, P);
    if (launched() != FFA_OK) return FFA_ERR_LAUNCH;
    const long long units = lines * (NCH + NCH / NB);
    hipLaunchKernelGGL(ffa_evict_move_kernel<NCH>, dim3((unsigned)((units + 3) / 4)), dim3(256), 0, st, P);
    return launched();
}

int launch_evict(const EvictParams& P, int head_dim, int elem_bytes, void* stream) {
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    switch (head_dim * elem_bytes / 16) {
        case 8: return evict_nch<8>(P, st);
        case 10: return evict_nch<10>(P, st);
        case 16: return evict_nch<16>(P, st);
        case 20: return evict_nch<20>(P, st);
        case 32: return evict_nch<32>(P, st);
        case 64: return evict_nch<64>(P, st);
        default: return FFA_ERR_HEAD_DIM;
    }
}

}  // namespace ffa
