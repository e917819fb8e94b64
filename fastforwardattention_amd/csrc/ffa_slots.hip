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
// A cache row of NCH 16-byte chunks is cut into column blocks of NB chunks (128 bytes; Dh = 80 has
// rows of 10 or 20 chunks: 5); an access of one wave to V covers 64 / NB slots of one block.
template <int NCH> struct Columns {
    static constexpr int NB = NCH % 8 == 0 ? 8 : 5;
    static constexpr int COLS = NCH / NB;
    static constexpr int RPI = 64 / NB;
};
// The wave of a workgroup of four, where the compiler sees that it is the same for all lanes.
__device__ __forceinline__ int wave_of_four() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6); }

// ---------------------------------------------------------------------------------------
// Commit.  One wave moves the accepted slots of one column block of one pair, K or V; path_len <= 64,
// so all of them are in its registers before the first is stored.  Bound by latency: a few KB a pair.
__device__ __forceinline__ void all_loaded() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

template <int NCH>
__global__ void __launch_bounds__(256) ffa_commit_kernel(const CommitParams P) {
    constexpr int NB = Columns<NCH>::NB, COLS = Columns<NCH>::COLS, RPI = Columns<NCH>::RPI;
    const int lane = threadIdx.x & 63;
    const unsigned unit = blockIdx.x * 4 + wave_of_four();
    const int pairs = P.B * P.H;
    const int col = (int)(unit % (2 * COLS));
    const unsigned rest = unit / (2 * COLS);
    const int pair = (int)(rest % pairs), cache = (int)(rest / pairs);
    if (cache >= P.n_caches) return;
    const int b = pair / P.H;
    const int base = P.lengths ? min(max(P.lengths[b], 0), P.t) : P.t;
    const int n = min(max(P.accepted[b], 0), P.path_len);
    if (n == 0) return;
    // Node of path entry `lane`: one that a group can have, and inside the cache, whatever the entry holds.
    const int entry = P.path[(size_t)b * P.path_len + min(lane, P.path_len - 1)];
    const int node = min(max(entry, 0), min(FFA_MAX_TREE_TOKENS, P.Lmax - base) - 1);
    const int c0 = (col >> 1) * NB;
    if ((col & 1) == 0) {
        u32x4_t* kc = static_cast<u32x4_t*>(P.k[cache]) + ((size_t)pair * NCH + c0) * P.Lmax + base;
        u32x4_t x[NB];
#pragma unroll
        for (int c = 0; c < NB; ++c) x[c] = (kc + (size_t)c * P.Lmax)[(unsigned)node];
        all_loaded();
        if (lane < n && node != lane) {
#pragma unroll
            for (int c = 0; c < NB; ++c) (kc + (size_t)c * P.Lmax)[(unsigned)lane] = x[c];
        }
    } else {
        u32x4_t* vc = static_cast<u32x4_t*>(P.v[cache]) + ((size_t)pair * P.Lmax + base) * NCH + c0;
        constexpr int IT = (64 + RPI - 1) / RPI;
        u32x4_t x[IT];
        const int r0 = lane / NB, c = lane % NB;
#pragma unroll
        for (int it = 0; it < IT; ++it) {
            x[it] = u32x4_t{0, 0, 0, 0};
            if (it * RPI >= n) break;
            const int row = it * RPI + r0, src = __shfl(node, min(row, 63));
            x[it] = vc[(unsigned)(src * NCH + c)];
        }
        all_loaded();
#pragma unroll
        for (int it = 0; it < IT; ++it) {
            if (it * RPI >= n) break;
            const int row = it * RPI + r0;
            if (r0 < RPI && row < n) vc[(unsigned)(row * NCH + c)] = x[it];
        }
    }
}

// ---------------------------------------------------------------------------------------
// Eviction, first kernel: which slots stay.  One workgroup a pair.  Weights become 32-bit keys in
// the order of the ranking, padding 0, NaN 1; a radix select over 8-bit digits finds the smallest
// key that stays and how many of its equals do; then the chosen slots are written in slot order,
// each behind the number chosen before it.  Up to held_slots() of a pair, all keys stay in
// registers; beyond, they are read again from the L2 by each of the up to five passes.
// A workgroup has as few waves, and its threads as few keys, as hold a pair's slots: every wave repeats the
// scan of a histogram, and every thread walks its keys, there or not (32 pairs of 1000 slots 9.2 us with 16
// waves, 9.4 us with 4 of 16 keys a thread, 6.6 us with 4 of 8; 512 pairs of 2256 slots 15.1 us with 16 of 8,
// 13.4 us with 4 of 16).
constexpr int held_slots(int waves, int keys) { return waves * 64 * keys; }

__device__ __forceinline__ uint32_t rank_key(float w) {
    if (w != w) return 1;
    const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.f);  // -0 ranks as +0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum over lanes 0 .. lane, in the vector pipeline (row shifts by 1, 2, 4, 8, then row broadcasts).
__device__ __forceinline__ unsigned wave_prefix(unsigned x) {
    x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, true);
    x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, true);
    x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, true);
    x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, true);
    x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, true);
    x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, true);
    return x;
}

// What stays of the ranked keys: all above `limit`, and the first `equal` of those that equal it.
struct Cut { uint32_t limit, equal; };

// One digit's step, by every wave for itself: finds the digit in which the `need`-th key from the
// top lies.  Returns whether the cut falls between two digits (all of that digit's keys stay).
__device__ __forceinline__ bool select_digit(const unsigned* hist, int lane, int shift, uint32_t* prefix, uint32_t* need) {
    // Counts from the top digit down: lane i holds digits 255 - 4 i .. 252 - 4 i.
    const u32x4_t q = *reinterpret_cast<const u32x4_t*>(&hist[252 - 4 * lane]);
    const unsigned n[4] = {q.w, q.z, q.y, q.x}, sum = (q.x + q.y) + (q.z + q.w);
    const unsigned incl = wave_prefix(sum);
    unsigned above = incl - sum, digit = 0, count = 0;
    const bool here = above < *need && incl >= *need;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const bool hit = count == 0 && above + n[e] >= *need;
        digit = hit ? 255 - 4 * lane - e : digit;
        above = count == 0 && !hit ? above + n[e] : above;
        count = hit ? n[e] : count;
    }
    const int from = __ffsll((unsigned long long)__ballot(here)) - 1;
    *prefix |= (uint32_t)__builtin_amdgcn_readlane((int)digit, from) << shift;
    *need -= (uint32_t)__builtin_amdgcn_readlane((int)above, from);
    return *need == (uint32_t)__builtin_amdgcn_readlane((int)count, from);
}

template <int NW, int KEYS>
__global__ void __launch_bounds__(NW * 64) ffa_evict_select_kernel(const EvictParams P) {
    // KEYS keys a thread in registers, or none: then they are read again.
    constexpr bool HELD = KEYS > 0;
    constexpr int R = HELD ? KEYS : 1, threads = NW * 64;
    __shared__ __align__(16) unsigned s_hist[4][256];
    __shared__ unsigned s_count[R * NW][2];  // chosen above the limit, equal to it: of each wave step (HELD) or wave
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int pairs = P.B * P.H;
    const int cache = blockIdx.x / pairs, pair = blockIdx.x % pairs, b = pair / P.H;
    const int length = P.lengths ? min(max(P.lengths[b], 0), P.t) : P.t;
    const int first = P.first_keys ? min(max(P.first_keys[b], 0), length) : 0;
    const float* w = P.w_src[cache] + (size_t)pair * P.src_len;
    float* to = P.w_dst[cache] + (size_t)pair * P.dst_len;
    int* kept = P.kept + ((size_t)cache * pairs + pair) * P.keep;
    const int tail = length - P.recent;  // slots from here on stay (if length > keep, which is >= recent)
    const int budget = P.keep - P.recent;

    if (length <= P.keep) {
        for (int j = tid; j < P.keep; j += threads) {
            kept[j] = j < length ? j : -1;
            if (j < length && to != w) to[j] = w[j];
        }
        return;
    }
    float held[R];
    if (HELD) {
#pragma unroll
        for (int r = 0; r < R; ++r) held[r] = r * threads + tid < length ? w[r * threads + tid] : 0.f;
    }
    auto key_of = [&](int j, float x) -> uint32_t { return j < first ? 0u : rank_key(x); };
    // body(slot, key) for this thread's ranked slots.
    auto each = [&](auto body) {
        if (HELD) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int j = r * threads + tid;
                if (j < tail) body(j, key_of(j, held[r]));
            }
        } else {
            for (int j = tid; j < tail; j += threads) body(j, key_of(j, w[j]));
        }
    };
    Cut cut = {0xffffffffu, 0};
    if (budget > 0) {
        for (int i = tid; i < 4 * 256; i += threads) s_hist[i / 256][i % 256] = 0;
        __syncthreads();
        uint32_t prefix = 0, need = budget;
        bool between = false;
        for (int d = 0; d < 4 && !between; ++d) {
            const int shift = 24 - 8 * d;
            each([&](int, uint32_t k) {
                if (d == 0 || ((k ^ prefix) >> (shift + 8)) == 0) atomicAdd(&s_hist[d][(k >> shift) & 255], 1u);
            });
            __syncthreads();
            between = select_digit(s_hist[d], lane, shift, &prefix, &need);
        }
        // Between two digits: everything from prefix on stays (prefix > 0, or all slots would).
        cut = between ? Cut{prefix - 1, 0} : Cut{prefix, need};
    }
    const unsigned long long below = (1ull << lane) - 1;
    if (HELD) {
        // Wave steps in slot order: step r * NW + wave.  At most 8192 in all: both counts in one word.
        unsigned long long m_more[R], m_equal[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int j = r * threads + tid;
            const uint32_t k = key_of(j, held[r]);
            m_more[r] = __ballot(j < tail && budget > 0 && k > cut.limit);
            m_equal[r] = __ballot(j < tail && budget > 0 && k == cut.limit);
            if (lane == 0) s_count[r * NW + wave][0] = (unsigned)__popcll(m_more[r]) << 16 | (unsigned)__popcll(m_equal[r]);
        }
        all_loaded();  // in place: nobody's weight is overwritten on its way here
        __syncthreads();
        const unsigned c0 = 2 * lane < R * NW ? s_count[2 * lane][0] : 0, c1 = 2 * lane < R * NW ? s_count[2 * lane + 1][0] : 0;
        const unsigned excl = wave_prefix(c0 + c1) - c0 - c1;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int j = r * threads + tid, step = r * NW + wave;
            const unsigned before = (unsigned)__builtin_amdgcn_readlane((int)excl, step / 2) +
                                    (step & 1 ? (unsigned)__builtin_amdgcn_readlane((int)c0, step / 2) : 0u);
            const unsigned more = (before >> 16) + __popcll(m_more[r] & below), equal = (before & 0xffff) + __popcll(m_equal[r] & below);
            int at = -1;
            if ((m_more[r] >> lane & 1) || ((m_equal[r] >> lane & 1) && equal < cut.equal)) at = (int)(more + min(equal, cut.equal));
            if (j >= tail && j < length) at = budget + j - tail;
            // Every weight is in a register by now: in place, nothing is lost.
            if (at >= 0) {
                kept[at] = j;
                to[at] = held[r];
            }
        }
        return;
    }
    // Stretches of whole wave steps, in slot order.
    const int steps = (tail + 64 * NW - 1) / (64 * NW);
    const int lo = wave * steps * 64, hi = min(lo + steps * 64, tail);
    unsigned more = 0, equal = 0;
    if (budget > 0) {
        for (int j0 = lo; j0 < hi; j0 += 64) {
            const int j = j0 + lane;
            const uint32_t k = j < hi ? key_of(j, w[j]) : 0;
            more += __popcll(__ballot(j < hi && k > cut.limit));
            equal += __popcll(__ballot(j < hi && k == cut.limit));
        }
    }
    if (lane == 0) {
        s_count[wave][0] = more;
        s_count[wave][1] = equal;
    }
    __syncthreads();
    more = equal = 0;
    for (int i = 0; i < wave; ++i) {
        more += s_count[i][0];
        equal += s_count[i][1];
    }
    if (budget > 0) {
        for (int j0 = lo; j0 < hi; j0 += 64) {
            const int j = j0 + lane;
            const uint32_t k = j < hi ? key_of(j, w[j]) : 0;
            const unsigned long long m_more = __ballot(j < hi && k > cut.limit);
            const unsigned long long m_equal = __ballot(j < hi && k == cut.limit);
            const unsigned e = equal + __popcll(m_equal & below);
            if ((m_more >> lane & 1) || ((m_equal >> lane & 1) && e < cut.equal))
                kept[more + __popcll(m_more & below) + min(e, cut.equal)] = j;
            more += __popcll(m_more);
            equal += __popcll(m_equal);
        }
    }
    for (int j = tid; j < P.recent; j += threads) kept[budget + j] = tail + j;
    __syncthreads();
    // Weights follow.  In place: a chunk's sources lie at or behind its targets, and behind the
    // targets of all chunks before it, so only the loads and stores of one chunk need the barrier.
    for (int j0 = 0; j0 < P.keep; j0 += threads) {
        const int j = j0 + tid;
        float x = 0.f;
        if (j < P.keep) x = w[kept[j]];
        all_loaded();
        __syncthreads();
        if (j < P.keep) to[j] = x;
    }
}

// Eviction, second kernel: the rows of K and V.  W waves take one chunk row of a pair's K (64
// slots of 16 bytes an access) or one column block of its V (128 bytes a slot) through the kept slots
// in order, a batch of W * 8 accesses at a time, the next one's loads in flight.  Where targets and sources are
// apart nothing orders the waves: W is 1, and a column is cut into segments.  In place, kept[j] >= j: what is
// stored for slots [j, j + n) can only overwrite sources of entries before j + n, so a batch is stored once
// all waves have its loads, and the loads of the next batch, whose sources are at j + n and after, need not wait
// for those stores.  No other workgroup touches the column.
// Bound by the memory: K is read in whole 128-byte lines of 8 slots, of which a random choice of slots
// leaves few out.
constexpr int kMoveBatch = 8;  // accesses of a batch

template <int NCH, int W>
__global__ void __launch_bounds__(W == 1 ? 256 : W * 64) ffa_evict_move_kernel(const EvictParams P) {
    constexpr int NB = Columns<NCH>::NB, COLS = Columns<NCH>::COLS, RPI = Columns<NCH>::RPI, U = kMoveBatch;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int pairs = P.B * P.H, cache = blockIdx.z;
    constexpr unsigned UNITS = NCH + COLS;
    const unsigned unit = blockIdx.x * 4 + wave;  // W == 1
    const int col = W == 1 ? (int)(unit % UNITS) : (int)blockIdx.y;
    const int pair = W == 1 ? (int)(unit / UNITS) : (int)blockIdx.x;
    if (pair >= pairs) return;
    const int b = pair / P.H;
    const int length = P.lengths ? min(max(P.lengths[b], 0), P.t) : P.t;
    const int stay = min(length, P.keep);
    const bool is_k = col < NCH;
    const char* src;
    char* dst;
    int rows, r0;               // slots of an access, this lane's slot
    unsigned step, lane_bytes;  // bytes between slots, of this lane's place in one
    if (is_k) {
        src = static_cast<const char*>(P.k_src[cache]) + ((size_t)pair * NCH + col) * P.src_len * 16;
        dst = static_cast<char*>(P.k_dst[cache]) + ((size_t)pair * NCH + col) * P.dst_len * 16;
        step = 16; rows = 64; r0 = lane; lane_bytes = 0;
    } else {
        src = static_cast<const char*>(P.v_src[cache]) + ((size_t)pair * P.src_len * NCH + (col - NCH) * NB) * 16;
        dst = static_cast<char*>(P.v_dst[cache]) + ((size_t)pair * P.dst_len * NCH + (col - NCH) * NB) * 16;
        step = NCH * 16; rows = RPI; r0 = lane / NB; lane_bytes = lane % NB * 16;
    }
    const bool in_place = W > 1 && src == dst;
    if (in_place && length <= P.keep) return;
    const int* kept = P.kept + ((size_t)cache * pairs + pair) * P.keep;
    const int batch = W * U * rows;
    if (W > 1) r0 += wave * rows;
    // Segments (W == 1) are whole batches.
    const int from0 = W == 1 ? blockIdx.y * P.segment_batches * batch : 0;
    const int end = W > 1 || blockIdx.y + 1 == gridDim.y ? stay : min(stay, from0 + P.segment_batches * batch);
    if (from0 >= end) return;

    int from[2][U];
    u32x4_t x[2][U];
    unsigned moved[2] = {0, 0};  // bit u: access u of the batch has a slot of this lane to store
    auto load_slots = [&](int s, int j0) {
#pragma unroll
        for (int u = 0; u < U; ++u) from[s][u] = kept[min(j0 + u * W * rows + r0, end - 1)];
    };
    auto load = [&](int s, int j0) {
        moved[s] = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + u * W * rows + r0;
            if (j < end && (is_k || lane < RPI * NB) && !(in_place && from[s][u] == j)) moved[s] |= 1u << u;
        }
        if (__any(moved[s] != 0)) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const size_t at = (size_t)from[s][u] * step + lane_bytes;
                x[s][u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(src + at));
            }
        }
    };
    auto store = [&](int s, int j0) {
        if (W > 1) {
            // The uses make the wave wait for this batch before it says so.
#pragma unroll
            for (int u = 0; u < U; ++u) asm volatile("" : "+v"(x[s][u]));
            __syncthreads();
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (moved[s] >> u & 1) {
                const size_t at = (size_t)(j0 + u * W * rows + r0) * step + lane_bytes;
                __builtin_nontemporal_store(x[s][u], reinterpret_cast<u32x4_t*>(dst + at));
            }
    };
    load_slots(0, from0);
    load_slots(1, from0 + batch);
    load(0, from0);
    for (int j0 = from0; j0 < end; j0 += 2 * batch) {
        load(1, j0 + batch);
        load_slots(0, j0 + 2 * batch);
        store(0, j0);
        load(0, j0 + 2 * batch);
        load_slots(1, j0 + 3 * batch);
        store(1, j0 + batch);
    }
}

// ---------------------------------------------------------------------------------------
static int launched() { return hipGetLastError() == hipSuccess ? FFA_OK : FFA_ERR_LAUNCH; }

template <int NCH> static int commit_nch(const CommitParams& P, hipStream_t st) {
    const long long units = (long long)P.n_caches * P.B * P.H * 2 * Columns<NCH>::COLS;
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

template <int NCH> static int evict_nch(EvictParams P, hipStream_t st) {
    const long long lines = (long long)P.n_caches * P.B * P.H;
    const dim3 grid((unsigned)lines);
    if (P.t <= held_slots(4, 4)) hipLaunchKernelGGL((ffa_evict_select_kernel<4, 4>), grid, dim3(4 * 64), 0, st, P);
    else if (P.t <= held_slots(4, 8)) hipLaunchKernelGGL((ffa_evict_select_kernel<4, 8>), grid, dim3(4 * 64), 0, st, P);
    else if (P.t <= held_slots(4, 16)) hipLaunchKernelGGL((ffa_evict_select_kernel<4, 16>), grid, dim3(4 * 64), 0, st, P);
    else if (P.t <= held_slots(16, 8)) hipLaunchKernelGGL((ffa_evict_select_kernel<16, 8>), grid, dim3(16 * 64), 0, st, P);
    else hipLaunchKernelGGL((ffa_evict_select_kernel<16, 0>), grid, dim3(16 * 64), 0, st, P);
    if (launched() != FFA_OK) return FFA_ERR_LAUNCH;
    constexpr int UNITS = NCH + Columns<NCH>::COLS;
    bool in_place = false;
    for (int i = 0; i < P.n_caches; ++i) in_place = in_place || P.k_src[i] == P.k_dst[i] || P.v_src[i] == P.v_dst[i];
    const int pairs = P.B * P.H, stay = P.t < P.keep ? P.t : P.keep;
    // In place: a column is one workgroup's, of 8 waves, or of 4 for few slots, where half of 8 would have none
    // of K's (us of the operator with 1, 4 and 8 waves, bf16: 8x32x128, 1000 of 1100 slots 71.0, 62.8, 64.7;
    // 1x32x64, 512 of 600 12.4, 9.5, 10.6; 8x32x128, 2048 of 4096 168, 146, 140; 1x8x128, 4283 of 5873 55.4, 27.0,
    // 24.6; 16 waves 25.5 there and 103 at 1000 of 1100).
    if (in_place) {
        const dim3 columns((unsigned)pairs, UNITS, (unsigned)P.n_caches);
        if (stay <= 1024) hipLaunchKernelGGL((ffa_evict_move_kernel<NCH, 4>), columns, dim3(256), 0, st, P);
        else hipLaunchKernelGGL((ffa_evict_move_kernel<NCH, 8>), columns, dim3(512), 0, st, P);
        return launched();
    }
    // Otherwise columns are cut where their waves would leave the chip half empty, down to one batch.
    const long long units = lines * UNITS;
    const int batches = (stay + kMoveBatch * Columns<NCH>::RPI - 1) / (kMoveBatch * Columns<NCH>::RPI);  // of V: K's hold more
    long long segments = (8192 + units - 1) / units;
    if (segments > batches) segments = batches < 1 ? 1 : batches;
    P.segment_batches = (int)((batches + segments - 1) / segments);
    if (P.segment_batches < 1) P.segment_batches = 1;
    hipLaunchKernelGGL((ffa_evict_move_kernel<NCH, 1>), dim3((unsigned)((pairs * UNITS + 3) / 4), (unsigned)segments, (unsigned)P.n_caches),
                       dim3(256), 0, st, P);
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
