// Device building blocks of the attention kernels (t2h_attn.hip,
// t2h_attn_bwd.hip): segments and their tiles, operand tiles in LDS, MFMA
// fragments.
//
// Every product is a 16x16x32 MFMA (f16 or bf16 operands, f32 sums). With h =
// lane / 16 and r = lane % 16, lane l holds of
//   A [16 x 32]  row r, k = 8h .. 8h+7       B [32 x 16]  column r, k = 8h .. 8h+7
//   C [16 x 16]  column r, rows 4h .. 4h+3
// A product's scores come out transposed, so that a lane holds one token of
// the side it keeps (column r) and four of the side that streams (rows 4h..).
// Two such C tiles (streaming tokens 0-15 and 16-31), rounded to 16 bits, are
// the B operand of the next product over 32 streaming tokens without any
// exchange between lanes, if that product counts its k so that slot (h, j)
// is streaming token 4h + j for j < 4 and 16 + 4h + j - 4 otherwise. Its A
// operand is the streaming tile transposed; ds_read_b64_tr_b16 reads it from
// the same LDS rows in just that order.
//
// A streaming tile lies in LDS as it does in memory, row by row (2 D bytes),
// with the 16-byte chunks of row t at slot c ^ swizzle(t). A row fragment
// reads chunk 4s + h of rows r; the LDS serves a 16-byte read in four turns
// of 16 lanes (0-3, 12-15, 20-27 / 4-11, 16-19, 28-31 / the same + 32). A
// transposed fragment reads 8 bytes of rows 4h + r/4, two chunks of eight rows
// for 32 lanes. The swizzle gives both distinct banks: over rows 0-7 (D = 128)
// its values are in different chunk pairs, and rows 4-11 and the others are
// each closed under a swap within the pairs.
#pragma once
#include "t2h_device.h"
#include "t2h_attn.h"

namespace t2h {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct AttnMma;
template <> struct AttnMma<_Float16> {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    typedef _Float16 v4 __attribute__((ext_vector_type(4)));
    __device__ static __forceinline__ f32x4 run(v8 a, v8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
template <> struct AttnMma<__bf16> {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    typedef __bf16 v4 __attribute__((ext_vector_type(4)));
    __device__ static __forceinline__ f32x4 run(v8 a, v8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};

// Block barrier that nothing is scheduled across; the caller has waited for
// what its wave reads or has written.
__device__ __forceinline__ void tile_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
}
// Wait until at most N of this wave's vector-memory operations are pending
// (gfx9 encoding: vmcnt[3:0] bits 3:0, vmcnt[5:4] bits 15:14).
template <int N>
__device__ __forceinline__ void wait_loads() {
    static_assert(N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}
__device__ __forceinline__ void wait_lds_reads() { __builtin_amdgcn_s_waitcnt(0xC07F); }   // lgkmcnt(0)

// ---- segments ---------------------------------------------------------------
// Row numbers are 32-bit (the entry points take no more rows); addresses are not.
struct Rows { int lo, hi; };
// Offset b, kept inside the tensor whatever it is.
__device__ __forceinline__ int offset_at(const int64_t* offsets, int rows, int b) {
    const int64_t o = offsets[b];
    return o < 0 ? 0 : o > rows ? rows : (int)o;
}
// Rows [lo, hi) of segment b: from the offsets, or equal shares.
__device__ __forceinline__ Rows segment_rows(const AttnSide& a, int b) {
    Rows s;
    if (a.offsets != nullptr) {
        s.lo = offset_at(a.offsets, a.rows, b);
        s.hi = offset_at(a.offsets, a.rows, b + 1);
        s.hi = s.hi < s.lo ? s.lo : s.hi;
    } else {
        s.lo = b * a.share;
        s.hi = s.lo + a.share;
    }
    return s;
}
// ... those of its keys that count.
__device__ __forceinline__ Rows segment_keys(const AttnArgs& a, int b) {
    Rows s = segment_rows(a.ks, b);
    if (a.k_lens != nullptr) {
        const int64_t n = a.k_lens[b] < 0 ? 0 : a.k_lens[b];
        if (n < s.hi - s.lo) s.hi = s.lo + (int)n;
    }
    return s;
}

// Number of segment b's first tile of BT rows: offsets[b] / BT + b, which leaves
// room for the ceil(length / BT) tiles of each segment, so a tile's segment is
// found by search and no prefix sum of tile counts is needed.
template <int BT>
__device__ __forceinline__ int first_tile(const AttnSide& a, int b) {
    return a.offsets != nullptr ? offset_at(a.offsets, a.rows, b) / BT + b : (a.share + BT - 1) / BT * b;
}
// Rows of tile t and its segment b; a number that no tile has comes back with lo
// >= hi. The 64 lanes look at 64 offsets at a time (all lanes active): a
// bisection waits for a load per halving, 6 us for 64 segments.
template <int BT>
__device__ __forceinline__ Rows tile_rows(const AttnSide& a, int nbatch, int t, int lane, int& b) {
    if (a.offsets != nullptr) {
        int lo = 0, n = nbatch;
        while (n > 1) {
            const int step = (n + 63) >> 6, i = lane * step;
            const uint64_t le = __ballot(i < n && first_tile<BT>(a, lo + (i < n ? i : 0)) <= t);
            const int k = le != 0 ? __popcll(le) - 1 : 0;
            lo += k * step;
            n = n - k * step < step ? n - k * step : step;
        }
        b = __builtin_amdgcn_readfirstlane(lo);
    } else {
        b = t / ((a.share + BT - 1) / BT);
    }
    Rows s = segment_rows(a, b);
    const int i = t - first_tile<BT>(a, b);
    s.lo = i < 0 || i > (s.hi - s.lo) / BT ? s.hi : s.lo + i * BT;
    return s;
}
// Tile numbers of a side (host).
inline int64_t tile_count(const AttnSide& a, int32_t nbatch, int bt) {
    if (a.offsets != nullptr) return a.rows / bt + nbatch;
    return (int64_t)((a.share + (int64_t)bt - 1) / bt) * nbatch;
}

// Logical number of physical block p of nb: contiguous ranges for the 8 XCDs
// (block p runs on XCD p % 8), so that the blocks one L2 serves at a time share
// a head's streaming side.
__device__ __forceinline__ int xcd_order(int p, int nb) {
    const int x = p & 7, i = p >> 3, q = nb >> 3, r = nb & 7;
    return x * q + (x < r ? x : r) + i;
}

// ---- tiles --------------------------------------------------------------------
template <int D>
__device__ __forceinline__ int swizzle(int t) {
    if constexpr (D == 128) return ((t & 7) << 1) ^ (((t >> 3) & 1) * 9);
    else return ((t >> 1 & 3) << 1) ^ (((t >> 3) & 1) * 5);
}

// (Not templates: hipcc's host pass drops a kernel template whose own body
// names these builtins.)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const uint8_t* p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ void rsrc_to_lds16(__amdgpu_buffer_rsrc_t r, uint8_t* lds, uint32_t off, uint32_t soff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, (int)off, (int)soff, 0, 0);
}
__device__ __forceinline__ void rsrc_to_lds4(__amdgpu_buffer_rsrc_t r, uint8_t* lds, uint32_t off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 4, (int)off, 0, 0, 0);
}
__device__ __forceinline__ u32x4 rsrc_load16(__amdgpu_buffer_rsrc_t r, uint32_t off) {
    return __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0);
}
typedef short s16x4 __attribute__((ext_vector_type(4)));
// (__restrict gives the read alias information of its own: without any, the
// compiler waits for every load to LDS in flight ahead of each of these. The
// kernels wait for the tiles they read themselves.)
__device__ __forceinline__ s16x4 lds_read_tr(const uint8_t* __restrict p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
}

// Bytes that a resource over n rows (at most BT) of 2 D bytes, stride bytes
// apart, covers: loads of rows past them return zeros, whatever memory holds there.
template <int D, int BT>
__device__ __forceinline__ uint32_t span_bytes(int n, uint32_t stride) {
    const int m = n < BT ? (n < 0 ? 0 : n) : BT;
    return m > 0 ? (uint32_t)(m - 1) * stride + D * 2 : 0;
}

// A [BT][D] tile of 16-bit rows copied to LDS by NW waves, 1 KB at a time.
template <int D, int BT, int NW> struct TileLoad {
    static constexpr int kBytes = BT * D * 2;
    static constexpr int kRowsPer = 512 / D;                 // rows of one wave's KB
    static constexpr int kLoads = kBytes / 1024 / NW;        // per wave
    static_assert(kBytes % (1024 * NW) == 0 && (kRowsPer * NW) % 16 == 0, "tile and waves");
    uint32_t off, stride;
    int wave;
    __device__ __forceinline__ void init(int wave_, int lane, int64_t row_stride) {
        wave = wave_;
        stride = (uint32_t)row_stride * 2;
        constexpr int kChunks = D / 8;
        const int t = wave * kRowsPer + lane / kChunks;
        off = (uint32_t)t * stride + (uint32_t)((lane % kChunks) ^ swizzle<D>(t & 15)) * 16;
    }
    // rows [row, row + BT) of the tensor at base, those from hi on as zeros
    __device__ __forceinline__ void issue(const uint8_t* base, int row, int hi, uint8_t* lds) const {
        const __amdgpu_buffer_rsrc_t r = rows_rsrc(base + (int64_t)row * stride, span_bytes<D, BT>(hi - row, stride));
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
            rsrc_to_lds16(r, lds + (i * NW + wave) * 1024, off, (uint32_t)(i * kRowsPer * NW) * stride);
    }
};

// A lane's addresses in a tile: row fragment s of 16-row tile i at
// (row ^ (s * 64)) + i * 32 D, transposed fragment of 16 columns c (elements
// 16 c ..) and streaming tokens 32 t .. at (tr ^ (c * 32)) + t * 64 D.
template <int D> struct FragAddr {
    int row, tr;
    __device__ __forceinline__ explicit FragAddr(int lane) {
        const int r = lane & 15, h = lane >> 4;
        row = r * (D * 2) + (h ^ swizzle<D>(r)) * 16;
        const int t = 4 * h + (r >> 2);
        tr = t * (D * 2) + ((((r & 3) >> 1) ^ swizzle<D>(t)) * 16) + (r & 1) * 8;
    }
};
template <typename T, int D>
__device__ __forceinline__ typename AttnMma<T>::v8 row_frag(const uint8_t* tile, int row, int i, int s) {
    return *reinterpret_cast<const typename AttnMma<T>::v8*>(tile + (row ^ (s * 64)) + i * (D * 32));
}
template <typename T, int D>
__device__ __forceinline__ typename AttnMma<T>::v8 tr_frag(const uint8_t* tile, int tr, int t, int c) {
    const uint8_t* p = tile + (tr ^ (c * 32)) + t * (D * 64);
    union { s16x4 h[2]; typename AttnMma<T>::v8 v; } u;
    u.h[0] = lds_read_tr(p);
    u.h[1] = lds_read_tr(p + D * 32);
    return u.v;
}

// A wave's own 16-token operand tile as B fragments, from memory: token r,
// elements 32 s + 8 h ..; tokens past n as zeros.
template <typename T, int D>
__device__ __forceinline__ void load_own(typename AttnMma<T>::v8 (&f)[D / 32], const uint8_t* base, int n,
                                         uint32_t stride, int lane) {
    const __amdgpu_buffer_rsrc_t r = rows_rsrc(base, span_bytes<D, 16>(n, stride));
    const uint32_t off = (uint32_t)(lane & 15) * stride + (uint32_t)(lane >> 4) * 16;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) f[s] = __builtin_bit_cast(typename AttnMma<T>::v8, rsrc_load16(r, off + s * 64));
}

// Two score tiles (streaming tokens 0-15 and 16-31) as one B operand.
template <typename T>
__device__ __forceinline__ typename AttnMma<T>::v8 pack_frag(const f32x4& a, const f32x4& b) {
    typename AttnMma<T>::v8 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = (T)a[i];
        v[4 + i] = (T)b[i];
    }
    return v;
}

template <int N>
__device__ __forceinline__ float sum_sq_all(const float (&x)[N]) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf(x[i], x[i], s);
    return s;
}

// What that rounding loses, rounded in turn: the two together hold twice the bits.
template <typename T>
__device__ __forceinline__ typename AttnMma<T>::v8 rest_frag(const f32x4& a, const f32x4& b,
                                                             const typename AttnMma<T>::v8& v) {
    typename AttnMma<T>::v8 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = (T)(a[i] - (float)v[i]);
        w[4 + i] = (T)(b[i] - (float)v[4 + i]);
    }
    return w;
}

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.69314718055994531f;
// 2^x: v_exp_f32 (results below 2^-126 are zero).
__device__ __forceinline__ float exp2_f(float x) { return __builtin_amdgcn_exp2f(x); }

}  // namespace
}  // namespace t2h
