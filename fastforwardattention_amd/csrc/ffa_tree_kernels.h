// Attention of a group of new tokens over the decode caches (gfx950, MFMA): drafted trees, chains,
// and the one-token step that sums attention weights.  Included by one translation unit per
// element type (ffa_tree_{f16,bf16,f32}.hip).
//
// Mathematics.  The rows of a (sample, cache head) pair are its tokens times its G query heads.
// For a tile of keys:  S^T = K Q^T (keys x rows),  P = 2^(S c - m),  O^T += V^T P^T (dims x rows),
// l += sum P, with c = softmax_scale * log2(e) and m one reference exponent a row.  Any m cancels
// in O / l, so m is only moved when a score exceeds it by `slack`: then rows are rescaled so that
// their largest P is 2^lift.  Pieces (waves, workgroups) are joined by their (m, l, O).
//
// Layout.  No operand passes through LDS.  A 16-byte chunk of a K cache row holds 8 (4) dims of
// one key, which is what one lane of a 16x16x32 (four 16x16x4) matrix product wants of its left
// operand.  The product's result has one row of Q a lane (lane % 16) and four keys in its
// registers, and the second product takes P in that order if V is read in it too: contraction
// slot (lane group g, j) is key 16 (j / 4) + 4 g + j % 4 of the tile.  V arrives in 16-byte (8-byte
// for Dh = 64) pieces of a key's row and is turned in registers, two 16-bit halves a v_perm.
//
// What bounds it: up to about 200 rows a pair in 16 bits the bytes of the caches (each read once a
// row block), above that the matrix units.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "ffa_cache_ops.h"
#include "ffa_device.h"

namespace ffa {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

// Scores may exceed a row's reference exponent by `slack`; a rescaled row starts at 2^lift.  In
// fp16 the range of P is what these two set: below 65504 at the top, and the smallest number, below which
// weights are dropped, is 2^-30 of the row's largest.  The other types' V has the exponents of the fp32 sums: there P
// stays below 4, so that the sums are finite where 4 times the sum of all |V| is.  (Lower, they would be finite for
// larger V, but the exponent's argument is rounded to 2^-24 of its size: at -29 that costs two bits of P.)
template <typename T> struct TreeRange { static constexpr float slack = 2.f, lift = -7.f; };
template <> struct TreeRange<uint16_t> { static constexpr float slack = 15.f, lift = 6.f; };

// Geometry of one element type, head dimension and number of row tiles.
template <typename T, int DH, int RT> struct TreeGeo {
    static constexpr int X = Elem<T>::X;                 // elements of a 16-byte chunk
    static constexpr int NCH = DH / X;                   // chunks of a row
    static constexpr int KK = (NCH + 3) / 4;             // chunk groups of a K row, one chunk a lane group
    static constexpr int NU = tree_tile_units(sizeof(T), DH, RT);  // 16-key matrix tiles of a wave tile
    static constexpr int TK = 16 * NU;                   // keys of a wave tile
    // A V row is cut into blocks of 16 * E dims, E of them a lane: E = 8 or 4 (16 or 8 bytes), the
    // last 16 dims of Dh = 80 one by one.
    static constexpr int E = X == 8 ? (DH >= 128 ? 8 : 4) : 4;
    static constexpr int NBLK = DH / (16 * E);           // whole blocks
    static constexpr int TAIL = DH - NBLK * 16 * E;      // 0, or 16
    static constexpr int DB = DH / 16;                   // 16-dim result tiles
};

// One chunk of K against one of Q for 16 keys x 16 rows.
__device__ __forceinline__ f32x4_t mma_qk(const uint4& k, const uint4& q, f32x4_t acc, uint16_t) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, k), __builtin_bit_cast(f16x8_t, q), acc, 0, 0, 0);
}
__device__ __forceinline__ f32x4_t mma_qk(const uint4& k, const uint4& q, f32x4_t acc, bf16_t) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, k), __builtin_bit_cast(bf16x8_t, q), acc, 0, 0, 0);
}
__device__ __forceinline__ f32x4_t mma_qk(const uint4& k, const uint4& q, f32x4_t acc, float) {
    const f32x4_t a = __builtin_bit_cast(f32x4_t, k), b = __builtin_bit_cast(f32x4_t, q);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], acc, 0, 0, 0);
    return acc;
}

// The weights of one row tile as right operands.  16-bit types: P = hi + lo, hi rounded towards zero, so
// that lo is not negative, lo to nearest: a weight is off by 2^-22 (fp16) or 2^-16 (bf16) of itself, or in fp16 by
// 2^-24, which is 2^-30 of the row's largest, whichever is more; the result's own rounding is to 11 or 8 bits.  Where hi is
// above zero lo is too: 0 * V would turn an infinite V into NaN.  Where hi is zero lo is zero: what has no weight,
// or is masked, adds nothing, however large its V.  (A NaN weight is NaN in hi, whatever lo is.)
struct PFrag16 { uint4 hi, lo; };
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void split_pair(float a, float b, uint32_t* hi, uint32_t* lo, uint16_t) {
    const uint32_t h = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
    *hi = h;
    // a - (lower half of h), b - (upper half): one instruction each, where the compiler converts first.
    float ra, rb;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(ra) : "v"(h), "v"(a));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(rb) : "v"(h), "v"(b));
    const u16x2_t rest = __builtin_bit_cast(u16x2_t, __builtin_convertvector(f32x2_t{ra, rb}, half2_t));
    // Neither part is negative: their bit patterns order as they do.  1 is 2^-24, the smallest fp16.
    u16x2_t one = {1, 1};
    asm("" : "+s"(one));  // a known 1 becomes two comparisons, five instructions in place of one
    const u16x2_t tiny = __builtin_elementwise_min(__builtin_bit_cast(u16x2_t, h), one);
    *lo = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(rest, tiny));
}
__device__ __forceinline__ void split_pair(float a, float b, uint32_t* hi, uint32_t* lo, bf16_t) {
    const uint32_t ua = __builtin_bit_cast(uint32_t, a), ub = __builtin_bit_cast(uint32_t, b);
    *hi = __builtin_amdgcn_perm(ub, ua, 0x07060302);
    const float la = a - __builtin_bit_cast(float, ua & 0xffff0000u), lb = b - __builtin_bit_cast(float, ub & 0xffff0000u);
    const u16x2_t rest = __builtin_bit_cast(u16x2_t, __builtin_convertvector(f32x2_t{la, lb}, bf16x2_t));
    // 0x0080 is 2^-126, the smallest normal number.
    const u16x2_t tiny = __builtin_elementwise_min(__builtin_bit_cast(u16x2_t, *hi), u16x2_t{0x0080, 0x0080});
    *lo = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(rest, tiny));
}

template <typename T> __device__ __forceinline__ PFrag16 split_weights(const float* p, T tag) {
    PFrag16 f;
    split_pair(p[0], p[1], &f.hi.x, &f.lo.x, tag);
    split_pair(p[2], p[3], &f.hi.y, &f.lo.y, tag);
    split_pair(p[4], p[5], &f.hi.z, &f.lo.z, tag);
    split_pair(p[6], p[7], &f.hi.w, &f.lo.w, tag);
    return f;
}

// ---------------------------------------------------------------------------------------
// V pieces of one wave tile, as loaded: piece j of a lane belongs to key 16 (j / 4) + 4 g + j % 4.
template <typename T, int DH, int RT> struct VTile {
    using G = TreeGeo<T, DH, RT>;
    static constexpr int NJ = 4 * G::NU;
    static constexpr int WORDS = G::E * (int)sizeof(T) / 4;     // 32-bit words of a piece: 2 or 4
    uint32_t w[NJ][G::NBLK][WORDS];
    uint32_t tail[G::TAIL ? NJ : 1];

    // STREAM: read once, past the caches' replacement order.
    template <bool STREAM> __device__ __forceinline__ void load(int j, const char* row, unsigned lane_row, int c) {
#pragma unroll
        for (int b = 0; b < G::NBLK; ++b) {
            const char* p = row + b * 16 * WORDS * 4 + (lane_row + (unsigned)c * (WORDS * 4));
            if constexpr (WORDS == 4) {
                const uint4 v = STREAM ? ld16(p) : *reinterpret_cast<const uint4*>(p);
                w[j][b][0] = v.x; w[j][b][1] = v.y; w[j][b][2] = v.z; w[j][b][3] = v.w;
            } else {
                typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
                const u32x2_t* at = reinterpret_cast<const u32x2_t*>(p);
                const u32x2_t v = STREAM ? __builtin_nontemporal_load(at) : *at;
                w[j][b][0] = v.x; w[j][b][1] = v.y;
            }
        }
        if constexpr (G::TAIL != 0) {
            const char* p = row + G::NBLK * 16 * G::E * (int)sizeof(T) + (lane_row + (unsigned)c * (unsigned)sizeof(T));
            if constexpr (sizeof(T) == 4) tail[j] = *reinterpret_cast<const uint32_t*>(p);
            else tail[j] = *reinterpret_cast<const uint16_t*>(p);
        }
    }
    // Key j holds nothing (a slot outside the sample's keys).
    __device__ __forceinline__ void clear(int j) {
#pragma unroll
        for (int b = 0; b < G::NBLK; ++b)
#pragma unroll
            for (int i = 0; i < WORDS; ++i) w[j][b][i] = 0;
        if constexpr (G::TAIL != 0) tail[j] = 0;
    }
    // Whether key j holds an infinity or NaN: the exponent's bits are all ones.
    static constexpr uint32_t kExponent = sizeof(T) == 4 ? 0x7f800000u : __is_same(T, bf16_t) ? 0x7f80u : 0x7c00u;
    __device__ __forceinline__ bool nonfinite(int j) const {
        uint32_t top = 0;  // largest magnitude; of both halves in 16-bit types
        auto word = [&](uint32_t x) {
            if constexpr (sizeof(T) == 4) top = max(top, x & 0x7fffffffu);
            else top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, top), __builtin_bit_cast(u16x2_t, x & 0x7fff7fffu)));
        };
#pragma unroll
        for (int b = 0; b < G::NBLK; ++b)
#pragma unroll
            for (int i = 0; i < WORDS; ++i) word(w[j][b][i]);
        if constexpr (G::TAIL != 0) word(tail[j]);
        if constexpr (sizeof(T) == 4) return top >= kExponent;
        else return (top & 0xffffu) >= kExponent || (top >> 16) >= kExponent;
    }
    // Infinities and NaN of key j become zero.
    __device__ __forceinline__ void drop_nonfinite(int j) {
        auto word = [](uint32_t x) -> uint32_t {
            if constexpr (sizeof(T) == 4) return (x & kExponent) == kExponent ? 0u : x;
            else return x & ((x & kExponent) == kExponent ? 0xffff0000u : 0xffffffffu) &
                        (((x >> 16) & kExponent) == kExponent ? 0x0000ffffu : 0xffffffffu);
        };
#pragma unroll
        for (int b = 0; b < G::NBLK; ++b)
#pragma unroll
            for (int i = 0; i < WORDS; ++i) w[j][b][i] = word(w[j][b][i]);
        if constexpr (G::TAIL != 0) tail[j] = word(tail[j]);
    }
    // Key j's pieces back to a row.
    __device__ __forceinline__ void store(int j, char* row, int c) const {
#pragma unroll
        for (int b = 0; b < G::NBLK; ++b) {
            char* p = row + (b * 16 + c) * (WORDS * 4);
            if constexpr (WORDS == 4) *reinterpret_cast<uint4*>(p) = make_uint4(w[j][b][0], w[j][b][1], w[j][b][2], w[j][b][3]);
            else *reinterpret_cast<uint2*>(p) = make_uint2(w[j][b][0], w[j][b][1]);
        }
        if constexpr (G::TAIL != 0) {
            char* p = row + (G::NBLK * 16 * G::E + c) * (int)sizeof(T);
            if constexpr (sizeof(T) == 4) *reinterpret_cast<uint32_t*>(p) = tail[j];
            else *reinterpret_cast<uint16_t*>(p) = (uint16_t)tail[j];
        }
    }
    // Left operand of result tile (block b, element e): keys 8 i .. 8 i + 7 of dim b * 16 E + c * E + e.
    __device__ __forceinline__ uint4 turned(int i, int b, int e) const {
        uint32_t o[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            if (b < G::NBLK) o[p] = __builtin_amdgcn_perm(w[8 * i + 2 * p + 1][b][e / 2], w[8 * i + 2 * p][b][e / 2], e % 2 ? 0x07060302 : 0x05040100);
            else o[p] = __builtin_amdgcn_perm(tail[G::TAIL ? 8 * i + 2 * p + 1 : 0], tail[G::TAIL ? 8 * i + 2 * p : 0], 0x05040100);
        }
        return make_uint4(o[0], o[1], o[2], o[3]);
    }
    __device__ __forceinline__ float at(int j, int b, int e) const {   // fp32
        return __builtin_bit_cast(float, b < G::NBLK ? w[j][b][e] : tail[G::TAIL ? j : 0]);
    }
};

template <typename T> __device__ __forceinline__ float load_elem(const T* p);
template <> __device__ __forceinline__ float load_elem(const uint16_t* p) { return (float)__builtin_bit_cast(_Float16, *p); }
template <> __device__ __forceinline__ float load_elem(const bf16_t* p) { return bf16_to_float(p->bits); }
template <> __device__ __forceinline__ float load_elem(const float* p) { return *p; }

// Four outputs, rounded once.
__device__ __forceinline__ void store_out4(uint16_t* to, const f32x4_t& o) {
    typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));
    *reinterpret_cast<f16x4_t*>(to) = __builtin_convertvector(o, f16x4_t);
}
__device__ __forceinline__ void store_out4(bf16_t* to, const f32x4_t& o) {
    typedef uint16_t u16x4_t __attribute__((ext_vector_type(4)));
    *reinterpret_cast<u16x4_t*>(to) = u16x4_t{float_to_bf16(o[0]), float_to_bf16(o[1]), float_to_bf16(o[2]), float_to_bf16(o[3])};
}
__device__ __forceinline__ void store_out4(float* to, const f32x4_t& o) { *reinterpret_cast<f32x4_t*>(to) = o; }

// n / d by the factor tree_magic(d).
__device__ __forceinline__ int quotient(int n, int d, unsigned magic) { return d == 1 ? n : (int)__umulhi((unsigned)n, magic); }

// Slots of sample b: [first, length).
__device__ __forceinline__ void sample_range(const int* first_keys, const int* lengths, int b, int t, int* first, int* length) {
    const int n = lengths ? min(max(lengths[b], 0), t) : t;
    *length = n;
    *first = first_keys ? min(max(first_keys[b], 0), n) : 0;
}

// Ancestors of node `lane`, itself included, as a bit mask, by one wave: the parent relation is
// squared six times (64 nodes are at most 63 steps from the root).
__device__ __forceinline__ uint64_t ancestor_mask(const int* parents, int tokens, int lane) {
    if (parents == nullptr) return lane == 63 ? ~0ull : (2ull << lane) - 1;
    int up = lane < tokens ? parents[lane] : -1;
    if (up < 0 || up >= lane) up = -1;
    uint32_t lo = lane < 32 ? 1u << lane : 0u, hi = lane < 32 ? 0u : 1u << (lane - 32);
#pragma unroll
    for (int s = 0; s < 6; ++s) {
        const int from = up < 0 ? lane : up;
        const uint32_t l2 = __shfl((int)lo, from), h2 = __shfl((int)hi, from);
        const int u2 = __shfl(up, from);
        lo |= l2;
        hi |= h2;
        up = up < 0 ? -1 : u2;
    }
    return ((uint64_t)hi << 32) | lo;
}

// ---------------------------------------------------------------------------------------
// Waves a SIMD that the registers are cut for.  Two hide a wave's loads and transcendentals behind the
// other's matrix products; what holds more than 256 registers of results and operands runs alone.
constexpr int tree_waves_per_simd(int dh, int rt) { return tree_two_waves(dh, rt) ? 2 : 1; }

// Q fragments of all row tiles, one register quadruple each: from 8 of them on they are read from LDS at
// every tile (128 cycles of it a wave at 16) and leave their registers to results and loads.  At 256 pairs
// of 8000 keys, in registers and in LDS: Dh 128, 64 rows 251 and 191 us (registers spilled), 32 rows 164
// and 155 us; Dh 64, 64 rows alike, at 1000 keys 25.3 and 23.6 us.
template <typename T, int DH, int RT> constexpr bool tree_q_in_lds() { return RT * TreeGeo<T, DH, RT>::KK >= 8; }
// Floats of LDS in front of the scores: the waves' results of one row tile, and Q.
template <int DH, int W> constexpr int tree_merge_floats() { return W * 16 * DH; }
template <typename T, int DH, int RT> constexpr int tree_q_floats() {
    return tree_q_in_lds<T, DH, RT>() ? RT * TreeGeo<T, DH, RT>::KK * 64 * 4 : 0;
}

// Arguments that the first loads need, ahead of the struct: they arrive in registers with the wave.
#define TREE_HOT_DECL const char *k_cache, const char *v_cache, int Lmax, int t, int n_splits, unsigned splits_magic, \
                      int tiles_per_split, int pieces, int ragged
#define TREE_HOT_OF(P) static_cast<const char*>((P).k_cache), static_cast<const char*>((P).v_cache), (P).Lmax, (P).t, \
                       (P).n_splits, (P).splits_magic, (P).tiles_per_split, (P).B * (P).H * (P).n_splits, \
                       (int)((P).lengths != nullptr || (P).first_keys != nullptr)

// STREAM: the caches are read once and go past the L2's replacement order, worth 13 % of a step over 1 GB.
// Not where several row blocks read the same keys (64 rows of Dh 256 in two blocks, 256 pairs of 8000
// keys: 585 us streamed, 548 us not; 96 rows of Dh 128 in two blocks, 16 pairs of 20000 keys: alike from
// HBM, 57 and 50 us where the last-level cache holds the keys).
template <typename T, int DH, int RT, int W, bool STREAM>
__global__ void __launch_bounds__(W * 64, tree_waves_per_simd(DH, RT)) ffa_tree_kernel(TREE_HOT_DECL, const TreeParams P) {
    using G = TreeGeo<T, DH, RT>;
    constexpr float kSlack = TreeRange<T>::slack, kLift = TreeRange<T>::lift;
    constexpr int NU = G::NU, TK = G::TK, KK = G::KK, NCH = G::NCH, DB = G::DB, NJ = 4 * NU;
    constexpr unsigned ROW = DH * sizeof(T);  // bytes of a cache row
    constexpr bool QLDS = tree_q_in_lds<T, DH, RT>();
    constexpr bool SHORT = RT == 1;           // few new tokens are likely: skip 16 keys that hold none
    extern __shared__ float4 s_dynamic[];
    f32x4_t* const s_acc = reinterpret_cast<f32x4_t*>(s_dynamic);                               // [W][DB][64]
    uint4* const s_q = reinterpret_cast<uint4*>(s_acc + W * DB * 64);                           // [RT][KK][64]
    float* const s_scores = reinterpret_cast<float*>(s_dynamic) + tree_merge_floats<DH, W>() + tree_q_floats<T, DH, RT>();  // [rows][score_lds]
    __shared__ float s_ml[W][RT * 16][2];  // a wave's m and l of a row; then s_ml[..][0] = its factor
    __shared__ float s_row[RT * 16][2];    // M and L of a row
    __shared__ uint64_t s_seen[64];
    __shared__ uint64_t s_bad[64 / TK];

    // Row blocks of one piece are 8 workgroups apart: the same XCD, whose L2 then holds the piece.
    const int rb = blockIdx.x / 8, piece = blockIdx.y * 8 + blockIdx.x % 8;
    if (piece >= pieces) return;
    const int pair = quotient(piece, n_splits, splits_magic), split = piece - pair * n_splits;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, c = lane & 15;
    const char* kc = k_cache + (size_t)pair * (unsigned)Lmax * ROW;
    const char* vc = v_cache + (size_t)pair * (unsigned)Lmax * ROW;

    int first = 0, length = t;
    if (ragged) sample_range(P.first_keys, P.lengths, quotient(pair, P.H, P.H_magic), t, &first, &length);

    // This wave's tiles: wave, wave + W, ... of the piece's cached keys, then its share of the tiles
    // of new tokens, which are dealt from the last wave on (the piece's shorter ends).
    const int piece0 = split * tiles_per_split * TK;
    const int lo = max(split * tiles_per_split, first / TK) + wave;
    const int hi = min((split + 1) * tiles_per_split, (length + TK - 1) / TK);
    const int n_cached = max(0, (hi - lo + W - 1) / W);

    uint4 kf[NU][KK];
    VTile<T, DH, RT> vt;
    // A chunk that does not exist (Dh = 80) must not hold an infinity against the zero of Q.
    auto existing = [&](const uint4& x, int kk) {
        if (NCH % 4 != 0 && kk == KK - 1 && kk * 4 + g >= NCH) return make_uint4(0, 0, 0, 0);
        return x;
    };
    // Loads of a tile: uniform addresses plus a 32-bit offset a lane.  Rows past `most` are read from it,
    // and masked.  In V of a whole tile of cached keys the rows are compile-time distances apart.
    auto load_cached_k = [&](int key0, int most) {
        const char* base = kc + (size_t)key0 * 16;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const int gg = NCH % 4 != 0 && kk == KK - 1 ? min(g, NCH - 1 - kk * 4) : g;
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                const char* p = base + (size_t)kk * 4 * (unsigned)Lmax * 16 + ((unsigned)gg * (unsigned)Lmax + (unsigned)min(u * 16 + c, most)) * 16u;
                kf[u][kk] = existing(STREAM ? ld16(p) : *reinterpret_cast<const uint4*>(p), kk);
            }
        }
    };
    auto load_whole_v = [&](int key0) {
        const char* base = vc + (size_t)key0 * ROW;
#pragma unroll
        for (int j = 0; j < NJ; ++j) vt.template load<STREAM>(j, base + ((j / 4) * 16 + j % 4) * ROW, (unsigned)g * 4u * ROW, c);
    };
    auto load_rows_v = [&](const char* base, unsigned step, int most) {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
            if (!SHORT || j / 4 * 16 <= most) vt.template load<STREAM>(j, base, (unsigned)min((j / 4) * 16 + g * 4 + j % 4, most) * step, c);
    };
    const bool begun = n_cached > 0 && lo * TK + TK <= length;
    if (begun) {
        load_cached_k(lo * TK, TK);
        load_whole_v(lo * TK);
    }

    // What the rest of the arguments say.
    const int b = quotient(pair, P.H, P.H_magic), h = pair - b * P.H;
    const int count = P.counts ? min(max(P.counts[b], 0), P.tokens) : P.tokens;
    const bool last = split == n_splits - 1;
    const char* kn = static_cast<const char*>(P.k) + (b * P.k_stride[0] + h * P.k_stride[1]) * (long long)sizeof(T);
    const char* vn = static_cast<const char*>(P.v) + (b * P.v_stride[0] + h * P.v_stride[1]) * (long long)sizeof(T);
    const unsigned kn_row = (unsigned)P.k_stride[2] * (unsigned)sizeof(T), vn_row = (unsigned)P.v_stride[2] * (unsigned)sizeof(T);
    const int row0 = rb * RT * 16;
    const int n_new = last ? max(0, ((count + TK - 1) / TK + wave) / W) : 0;
    const int n_tiles = n_cached + n_new;
    // Tile i of this wave: its first key, counted in the cache or among the new tokens.
    auto key0_of = [&](int i) { return (i < n_cached ? lo + i * W : W - 1 - wave + (i - n_cached) * W) * TK; };
    auto load_k = [&](int i) {
        const int key0 = key0_of(i);
        if (i < n_cached) {
            load_cached_k(key0, length - 1 - key0);
        } else {
            const char* base = kn + (size_t)key0 * kn_row;
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                if (SHORT && key0 + u * 16 >= count) break;
                const unsigned row = (unsigned)min(u * 16 + c, count - 1 - key0) * kn_row;
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) kf[u][kk] = existing(ld16(base + (row + (unsigned)min(kk * 4 + g, NCH - 1) * 16u)), kk);
            }
        }
    };
    auto load_v = [&](int i) {
        const int key0 = key0_of(i);
        if (i < n_cached && key0 + TK <= length) load_whole_v(key0);
        else if (i < n_cached) load_rows_v(vc + (size_t)key0 * ROW, ROW, length - 1 - key0);
        else load_rows_v(vn + (size_t)key0 * vn_row, vn_row, count - 1 - key0);
    };
    if (!begun && n_tiles > 0) {
        load_k(0);
        load_v(0);
    }

    // Lane i of a wave that has new tokens: node i's ancestors.
    uint64_t ancestors = 0;
    if (n_new > 0) {
        ancestors = ancestor_mask(P.parents ? P.parents + (size_t)b * P.tokens : nullptr, P.tokens, lane);
        if (wave == W - 1) s_seen[lane] = ancestors;
    }

    // Q: chunk kk * 4 + g of row row0 + rt * 16 + c; rows and chunks that do not exist are zero.
    // The factor of the scores is positive: a negative softmax_scale turns Q's sign.
    auto load_q = [&](int rt, int kk) {
        const int row = row0 + rt * 16 + c, ch = kk * 4 + g;
        const int token = quotient(row, P.G, P.G_magic), gh = row - token * P.G;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (row < P.rows && ch < NCH && P.q_sign != 0) {
            constexpr uint32_t sign = sizeof(T) == 4 ? 0x80000000u : 0x80008000u;
            const uint32_t turn = P.q_sign < 0 ? sign : 0u;
            x = *reinterpret_cast<const uint4*>(static_cast<const char*>(P.q) + ch * 16 +
                                                (b * P.q_stride[0] + (long long)(h * P.G + gh) * P.q_stride[1] + token * P.q_stride[2]) * (long long)sizeof(T));
            x.x ^= turn; x.y ^= turn; x.z ^= turn; x.w ^= turn;
        }
        return x;
    };
    uint4 qf[QLDS ? 1 : RT][QLDS ? 1 : KK];
    if constexpr (QLDS) {
        for (int i = wave; i < RT * KK; i += W) s_q[i * 64 + lane] = load_q(i / KK, i % KK);
        __syncthreads();
    } else {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) qf[rt][kk] = load_q(rt, kk);
    }

    f32x4_t acc[RT][DB];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -INFINITY;
        l[rt] = 0.f;
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[rt][db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    for (int i = 0; i < n_tiles; ++i) {
        const int key0 = key0_of(i);
        const bool cached = i < n_cached;
        const bool masked = !cached || key0 < first || key0 + TK > length;
        // New tokens are appended from the registers that hold them; nobody reads cache slots from
        // `length` on.
        if (!cached && rb == 0) {
            char* kw = const_cast<char*>(kc);
            char* vw = const_cast<char*>(vc);
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                if (SHORT && key0 + u * 16 >= count) break;
                const int node = key0 + u * 16 + c;
#pragma unroll
                for (int kk = 0; kk < KK; ++kk)
                    if (node < count && kk * 4 + g < NCH) st16(kw + ((size_t)(kk * 4 + g) * Lmax + length + node) * 16, kf[u][kk]);
            }
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                if (SHORT && key0 + j / 4 * 16 >= count) break;
                const int node = key0 + (j / 4) * 16 + g * 4 + j % 4;
                if (node < count) vt.store(j, vw + (size_t)(length + node) * ROW, c);
            }
        }
        if constexpr (QLDS) asm volatile("" ::: "memory");  // Q stays in LDS: its registers are wanted
        f32x4_t s[RT][NU];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                s[rt][u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kk = 0; kk < KK; ++kk)
                    s[rt][u] = mma_qk(kf[u][kk], QLDS ? s_q[(rt * KK + kk) * 64 + lane] : qf[QLDS ? 0 : rt][QLDS ? 0 : kk], s[rt][u], T{});
            }
        if (i + 1 < n_tiles) load_k(i + 1);
        if (masked) {
            // Bit j: this lane's key j is seen.  Cached keys: the sample's range; new ones: ancestors.
            auto bits_of = [&](uint64_t range) {
                uint32_t x = 0;
#pragma unroll
                for (int u = 0; u < NU; ++u) x |= ((uint32_t)(range >> (u * 16 + g * 4)) & 15u) << (4 * u);
                return x;
            };
            uint64_t range = 0;
            if (cached) {
                const int from = min(max(first - key0, 0), TK), to = min(length - key0, TK);
                range = (to == 64 ? ~0ull : (1ull << to) - 1) & (from == 64 ? 0ull : ~0ull << from);
            }
            uint32_t held = cached ? bits_of(range) : 0;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                uint32_t bits = held;
                if (!cached) {
                    const int row = row0 + rt * 16 + c, token = min(quotient(row, P.G, P.G_magic), 63);
                    const uint64_t of_row = (uint64_t)(uint32_t)__shfl((int)(ancestors >> 32), token) << 32 | (uint32_t)__shfl((int)ancestors, token);
                    bits = row < P.rows ? bits_of(of_row >> key0) : 0u;
                }
#pragma unroll
                for (int j = 0; j < NJ; ++j)
                    if (!(bits >> j & 1)) s[rt][j / 4][j % 4] = -INFINITY;
            }
            // V of what no row sees must not meet a zero weight: 0 * NaN.  An infinite or NaN value of a
            // new token is added at the end, to the rows that see it.
            if (cached) {
#pragma unroll
                for (int j = 0; j < NJ; ++j)
                    if (!(held >> j & 1)) vt.clear(j);
            } else {
                bool any = false;
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    if (key0 + (j / 4) * 16 + g * 4 + j % 4 >= count) vt.clear(j);
                    if (!SHORT || key0 + j / 4 * 16 < count) any |= vt.nonfinite(j);
                }
                uint64_t bad = 0;
                if (__any(any)) {
#pragma unroll
                    for (int j = 0; j < NJ; ++j) {
                        const uint64_t who = __ballot(vt.nonfinite(j));
                        vt.drop_nonfinite(j);
#pragma unroll
                        for (int w = 0; w < 4; ++w) bad |= (who >> (16 * w) & 0xffff) != 0 ? 1ull << ((j / 4) * 16 + w * 4 + j % 4) : 0ull;
                    }
                }
                if (lane == 0) s_bad[key0 / TK] = bad;
            }
        }
        if (P.ws_scores != nullptr) {
            // In LDS if the piece's fit (key - first key of the piece), else in the workspace; the new
            // token's scores lie in the last 64 words.
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const int row = row0 + rt * 16 + c;
                if (row < P.rows) {
                    f32x4_t x[NU];
#pragma unroll
                    for (int u = 0; u < NU; ++u) x[u] = s[rt][u] * P.scale_log2e;
                    if (P.score_lds != 0) {
                        float* to = s_scores + row * P.score_lds + (cached ? key0 - piece0 : P.score_lds - 64) + g * 4;
#pragma unroll
                        for (int u = 0; u < NU; ++u) *reinterpret_cast<f32x4_t*>(to + u * 16) = x[u];
                    } else {
                        float* to = P.ws_scores + ((size_t)pair * P.rows + row) * P.score_stride + (cached ? key0 : P.score_stride - 64) + g * 4;
#pragma unroll
                        for (int u = 0; u < NU; ++u) *reinterpret_cast<f32x4_t*>(to + u * 16) = x[u];
                    }
                }
            }
        }
        constexpr int NP = sizeof(T) == 2 ? NU / 2 : 1;  // right operands of 32 keys
        PFrag16 pf[RT][NP];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float x[NJ];
            float top = s[rt][0][0];
#pragma unroll
            for (int j = 1; j < NJ; ++j) top = fmaxf(top, s[rt][j / 4][j % 4]);
            top *= P.scale_log2e;
            if (__any(top > m[rt] + kSlack)) {
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const float to = top > m[rt] + kSlack ? top - kLift : m[rt];
                const float f = to == m[rt] ? 1.f : __builtin_amdgcn_exp2f(m[rt] - to);
                m[rt] = to;
                l[rt] *= f;
#pragma unroll
                for (int db = 0; db < DB; ++db) acc[rt][db] *= f;
            }
            const float ref = m[rt] == -INFINITY ? 0.f : -m[rt];
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                x[j] = __builtin_amdgcn_exp2f(fmaf(s[rt][j / 4][j % 4], P.scale_log2e, ref));
                sum += x[j];
            }
            l[rt] += sum;
            if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int q = 0; q < NP; ++q) pf[rt][q] = split_weights(x + 8 * q, T{});
            } else {
#pragma unroll
                for (int j = 0; j < NJ; ++j) s[rt][j / 4][j % 4] = x[j];
            }
        }
        // Turned ahead of the products, V leaves its registers to the next tile's loads: 8 % of a step over
        // 1000 keys.  Where registers are short it costs more than that (four row tiles of Dh 128: -6 %).
        constexpr bool EARLY = sizeof(T) == 2 && RT <= 2 && DH <= 128;
        uint4 tv[EARLY ? NP : 1][EARLY ? DB : 1];
        if constexpr (EARLY) {
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int q = 0; q < NP; ++q) tv[q][db] = vt.turned(q, db < G::NBLK * G::E ? db / G::E : G::NBLK, db < G::NBLK * G::E ? db % G::E : 0);
            if (i + 1 < n_tiles) load_v(i + 1);
        }
#pragma unroll
        for (int db = 0; db < DB; ++db) {
            const int blk = db < G::NBLK * G::E ? db / G::E : G::NBLK, e = db < G::NBLK * G::E ? db % G::E : 0;
            if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int q = 0; q < NP; ++q) {
                    const uint4 a = EARLY ? tv[EARLY ? q : 0][EARLY ? db : 0] : vt.turned(q, blk, e);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        acc[rt][db] = mma_qk(a, pf[rt][q].hi, acc[rt][db], T{});
                        acc[rt][db] = mma_qk(a, pf[rt][q].lo, acc[rt][db], T{});
                    }
                }
            } else {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
                        acc[rt][db] = __builtin_amdgcn_mfma_f32_16x16x4f32(vt.at(j, blk, e), s[rt][j / 4][j % 4], acc[rt][db], 0, 0, 0);
            }
        }
        if (!EARLY && i + 1 < n_tiles) load_v(i + 1);
    }

    // ---- join the waves: out = sum_w O_w 2^(m_w - M) / sum_w l_w 2^(m_w - M) ----
    // Four dims that lie side by side are one item; a lane has DB of them a row tile.  The items go
    // through LDS in the lanes' own order, so that neither side meets a bank conflict.
    auto put = [&](int rt) {
        f32x4_t* to = s_acc + wave * DB * 64 + lane;
#pragma unroll
        for (int it = 0; it < DB; ++it) {
            if (it < G::NBLK * G::E) {
                constexpr int Q4 = G::E / 4;
                const int db = it / G::E * G::E + it % Q4 * 4, r = it % G::E / Q4;
                to[it * 64] = f32x4_t{acc[rt][db][r], acc[rt][db + 1][r], acc[rt][db + 2][r], acc[rt][db + 3][r]};
            } else {
                to[it * 64] = acc[rt][it];
            }
        }
    };
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        float sum = l[rt];
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        if (g == 0) {
            s_ml[wave][rt * 16 + c][0] = m[rt];
            s_ml[wave][rt * 16 + c][1] = sum;
        }
    }
    put(0);
    __syncthreads();
    const bool whole = n_splits == 1, weights = P.ws_scores != nullptr;
    if (tid < RT * 16) {
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) M = fmaxf(M, s_ml[w][tid][0]);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float mw = s_ml[w][tid][0];
            const float f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - M);
            L += f * s_ml[w][tid][1];
            s_ml[w][tid][0] = f;
        }
        s_row[tid][0] = M;
        s_row[tid][1] = L;
        const int row = row0 + tid;
        if ((!whole || weights) && row < P.rows) {
            float* to = P.ws_ml + (((size_t)pair * n_splits + split) * P.rows + row) * 2;
            // A maximum of -infinity says that the piece holds nothing; one of NaN scores alone has that too.
            to[0] = M == -INFINITY && L != 0.f ? 0.f : M;
            to[1] = L;
        }
    }
    uint64_t bad = 0;
    if (last) {
#pragma unroll
        for (int d = 0; d < 64 / TK; ++d)
            if (d * TK < count) bad |= s_bad[d] << (d * TK);
    }
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        if (rt > 0) {
            __syncthreads();
            put(rt);
            __syncthreads();
        }
        for (int i = tid; i < DB * 64; i += W * 64) {
            const int it = i / 64, r = i % 16, gg = i / 16 % 4;
            const int row = row0 + rt * 16 + r;
            if (row >= P.rows) continue;
            constexpr int Q4 = G::E / 4;
            const int d = it < G::NBLK * G::E ? it / G::E * 16 * G::E + (gg * 4 + it % G::E / Q4) * G::E + it % Q4 * 4
                                              : G::NBLK * 16 * G::E + gg * 4;
            f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < W; ++w) o += s_acc[w * DB * 64 + i] * s_ml[w][rt * 16 + r][0];
            const int token = quotient(row, P.G, P.G_magic);
            if (bad != 0) {
                for (uint64_t todo = bad & s_seen[token]; todo != 0; todo &= todo - 1) {
                    const int node = __ffsll((unsigned long long)todo) - 1;
                    const T* vr = reinterpret_cast<const T*>(vn + node * vn_row) + d;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = load_elem(vr + e);
                        if (!__builtin_isfinite(x)) o[e] += x;
                    }
                }
            }
            if (!whole) {
                *reinterpret_cast<f32x4_t*>(P.ws_acc + (((size_t)pair * n_splits + split) * P.rows + row) * DH + d) = o;
            } else if (token < count || P.zero_rest) {
                T* to = static_cast<T*>(P.out) + b * P.out_stride[0] + (long long)(h * P.G + row - token * P.G) * P.out_stride[1] + token * P.out_stride[2];
                store_out4(to + d, token < count ? o / s_row[rt * 16 + r][1] : f32x4_t{0.f, 0.f, 0.f, 0.f});
            }
        }
    }

    // ---- weight-summing step with scores in LDS (one row tile): the weights if this piece is all there
    // is, else the scores go to the workspace, where the pieces' kernel finds them ----
    if (weights && P.score_lds != 0) {
        const int from = max(first, piece0), to = min(length, piece0 + tiles_per_split * TK);
        if (whole) {
            // Eight keys a thread and step: their sums are on the way while the weights are formed.
            float* kw = P.key_weights + (size_t)pair * Lmax;
            constexpr int U = 8;
            for (int j0 = from + tid; j0 <= to; j0 += U * W * 64) {
                float sum[U], w[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    sum[u] = kw[min(j0 + u * W * 64, to)];
                    w[u] = 0.f;
                }
                for (int r = 0; r < P.rows; ++r) {
                    const float M = s_row[r][0], per = 1.f / s_row[r][1];
                    const float* x = s_scores + r * P.score_lds;
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const int j = min(j0 + u * W * 64, to);
                        w[u] += __builtin_amdgcn_exp2f(x[j == length ? P.score_lds - 64 : j - piece0] - M) * per;
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int j = j0 + u * W * 64;
                    if (j <= to) kw[j] = j == length ? w[u] : sum[u] + w[u];
                }
            }
        } else {
            for (int r = 0; r < P.rows; ++r) {
                float* ws = P.ws_scores + ((size_t)pair * P.rows + r) * P.score_stride;
                for (int j = from + tid; j < to; j += W * 64) ws[j] = s_scores[r * P.score_lds + j - piece0];
                if (last && tid == 0) ws[P.score_stride - 64] = s_scores[r * P.score_lds + P.score_lds - 64];
            }
        }
    }
}

// After the pieces, a pair a grid row.  The first join_blocks workgroups of a pair join its rows, four
// dims a thread: out = sum_i O_i 2^(m_i - M) / sum_i l_i 2^(m_i - M).  The others turn scores into weights,
// 1024 keys each.  Bound by latency (the partial results are a few MB at most): what the loads need comes
// in the leading arguments, and eight pieces' loads are in flight at a time.
struct RowTotal { float M, L; };
// By a whole wave: lane s takes pieces s and s + 64 (there are at most 128).
__device__ __forceinline__ RowTotal row_total(const float* ws_ml, size_t slot0, int n_splits, int rows, int lane) {
    float m[2], l[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int s = lane + 64 * i;
        const size_t at = (slot0 + (size_t)min(s, n_splits - 1) * rows) * 2;
        m[i] = s < n_splits ? ws_ml[at] : -INFINITY;
        l[i] = s < n_splits ? ws_ml[at + 1] : 0.f;
    }
    const float M = wave_max(fmaxf(m[0], m[1]));
    float L = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) L += m[i] == -INFINITY ? 0.f : l[i] * __builtin_amdgcn_exp2f(m[i] - M);
    return {M, wave_sum(L)};
}

constexpr int kFinishKeys = 4;  // keys a thread

template <typename T, int DH>
__global__ void __launch_bounds__(256) ffa_tree_finish_kernel(const float* ws_acc, const float* ws_ml, int n_splits, int rows,
                                                              int join_blocks, const TreeParams P) {
    const int pairs = P.B * P.H;
    for (int pair = blockIdx.y; pair < pairs; pair += gridDim.y) {
        if ((int)blockIdx.x < join_blocks) {
            const int i = blockIdx.x * 256 + threadIdx.x;
            const int row = i / (DH / 4), d = i % (DH / 4) * 4;
            if (row >= rows) return;
            const size_t slot0 = (size_t)pair * n_splits * rows + row;
            constexpr int U = 8;
            float M = -INFINITY, L = 0.f;
            f32x4_t o = {0.f, 0.f, 0.f, 0.f};
            for (int s0 = 0; s0 < n_splits; s0 += U) {
                f32x2_t ml[U];
                f32x4_t os[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const size_t slot = slot0 + (size_t)min(s0 + u, n_splits - 1) * rows;
                    ml[u] = *reinterpret_cast<const f32x2_t*>(ws_ml + slot * 2);
                    os[u] = *reinterpret_cast<const f32x4_t*>(ws_acc + slot * DH + d);
                }
                float top = M;
#pragma unroll
                for (int u = 0; u < U; ++u) top = s0 + u < n_splits ? fmaxf(top, ml[u].x) : top;
                const float back = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - top);
                L = M == -INFINITY ? 0.f : L * back;
                o = M == -INFINITY ? f32x4_t{0.f, 0.f, 0.f, 0.f} : o * back;
                M = top;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const bool counts = s0 + u < n_splits && ml[u].x != -INFINITY;
                    const float f = counts ? __builtin_amdgcn_exp2f(ml[u].x - M) : 0.f;
                    L += counts ? ml[u].y * f : 0.f;
                    o += counts ? os[u] * f : f32x4_t{0.f, 0.f, 0.f, 0.f};
                }
            }
            const int b = quotient(pair, P.H, P.H_magic), h = pair - b * P.H, token = quotient(row, P.G, P.G_magic);
            const bool there = P.counts == nullptr || token < P.counts[b];
            if (there || P.zero_rest) {
                T* to = static_cast<T*>(P.out) + b * P.out_stride[0] + (long long)(h * P.G + row - token * P.G) * P.out_stride[1] + token * P.out_stride[2];
                store_out4(to + d, there ? o / L : f32x4_t{0.f, 0.f, 0.f, 0.f});
            }
            continue;
        }
        int first, length;
        sample_range(P.first_keys, P.lengths, quotient(pair, P.H, P.H_magic), P.t, &first, &length);
        const int j0 = (blockIdx.x - join_blocks) * 256 * kFinishKeys + threadIdx.x;
        float w[kFinishKeys] = {};
        for (int row = 0; row < rows; ++row) {
            const float* x = P.ws_scores + ((size_t)pair * rows + row) * P.score_stride;
            float z[kFinishKeys];
#pragma unroll
            for (int k = 0; k < kFinishKeys; ++k) {
                const int j = j0 + k * 256;
                z[k] = j > length || j < first ? -INFINITY : x[j == length ? P.score_stride - 64 : j];
            }
            const RowTotal t = row_total(ws_ml, (size_t)pair * n_splits * rows + row, n_splits, rows, threadIdx.x & 63);
#pragma unroll
            for (int k = 0; k < kFinishKeys; ++k) w[k] += __builtin_amdgcn_exp2f(z[k] - t.M) / t.L;
        }
#pragma unroll
        for (int k = 0; k < kFinishKeys; ++k) {
            const int j = j0 + k * 256;
            float* to = P.key_weights + (size_t)pair * P.Lmax + j;
            if (j == length) *to = w[k];
            else if (j < length && j >= first) *to += w[k];
        }
    }
}

// ---------------------------------------------------------------------------------------
template <typename T, int DH, int RT, int W> int launch_tree_kernel(const TreeParams& P, hipStream_t st) {
    const dim3 grid(8u * (unsigned)P.row_blocks, (unsigned)((P.B * P.H * P.n_splits + 7) / 8));
    const size_t lds = (size_t)(tree_merge_floats<DH, W>() + tree_q_floats<T, DH, RT>() + P.rows * P.score_lds) * sizeof(float);
    // With one row tile there are several row blocks on few keys only, where it makes no difference.
    if (RT > 1 && P.row_blocks > 1) hipLaunchKernelGGL((ffa_tree_kernel<T, DH, RT, W, (RT == 1)>), grid, dim3(W * 64), lds, st, TREE_HOT_OF(P), P);
    else hipLaunchKernelGGL((ffa_tree_kernel<T, DH, RT, W, true>), grid, dim3(W * 64), lds, st, TREE_HOT_OF(P), P);
    return hipGetLastError() == hipSuccess ? FFA_OK : FFA_ERR_LAUNCH;
}

template <typename T, int DH> int launch_tree_dh(const TreeParams& P, const TreePlan& plan, hipStream_t st) {
    int rc = FFA_ERR_PLAN;
    if (plan.waves > 4) {
        if constexpr (tree_wide(DH, 1))
            if (plan.row_tiles == 1) rc = launch_tree_kernel<T, DH, 1, 8>(P, st);
        if constexpr (tree_wide(DH, 2))
            if (plan.row_tiles == 2) rc = launch_tree_kernel<T, DH, 2, 8>(P, st);
        if constexpr (tree_wide(DH, 3))
            if (plan.row_tiles == 3) rc = launch_tree_kernel<T, DH, 3, 8>(P, st);
        if constexpr (tree_wide(DH, 4))
            if (plan.row_tiles == 4) rc = launch_tree_kernel<T, DH, 4, 8>(P, st);
    } else {
        if (plan.row_tiles == 1) rc = launch_tree_kernel<T, DH, 1, 4>(P, st);
        if constexpr (tree_row_tiles(DH) > 1)
            if (plan.row_tiles == 2) rc = launch_tree_kernel<T, DH, 2, 4>(P, st);
        if constexpr (tree_row_tiles(DH) > 2)
            if (plan.row_tiles == 3) rc = launch_tree_kernel<T, DH, 3, 4>(P, st);
        if constexpr (tree_row_tiles(DH) > 3)
            if (plan.row_tiles == 4) rc = launch_tree_kernel<T, DH, 4, 4>(P, st);
    }
    if (rc != FFA_OK) return rc;
    const bool weights = P.ws_scores != nullptr && (P.n_splits > 1 || P.score_lds == 0);
    if (P.n_splits > 1 || weights) {
        const int join_blocks = P.n_splits > 1 ? (int)(((long long)P.rows * (DH / 4) + 255) / 256) : 0;
        const int key_blocks = weights ? (P.t + 256 * kFinishKeys) / (256 * kFinishKeys) : 0, pairs = P.B * P.H;
        const dim3 grid((unsigned)(join_blocks + key_blocks), (unsigned)(pairs < 65535 ? pairs : 65535));
        hipLaunchKernelGGL((ffa_tree_finish_kernel<T, DH>), grid, dim3(256), 0, st, P.ws_acc, P.ws_ml, P.n_splits, P.rows, join_blocks, P);
        if (hipGetLastError() != hipSuccess) return FFA_ERR_LAUNCH;
    }
    return FFA_OK;
}

template <typename T> int launch_tree_type(const TreeParams& P, int head_dim, const TreePlan& plan, void* stream) {
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    switch (head_dim) {
        case 64: return launch_tree_dh<T, 64>(P, plan, st);
        case 80: return launch_tree_dh<T, 80>(P, plan, st);
        case 128: return launch_tree_dh<T, 128>(P, plan, st);
        case 256: return launch_tree_dh<T, 256>(P, plan, st);
        default: return FFA_ERR_HEAD_DIM;
    }
}

}  // namespace ffa
