// Backward pass of the attention (t2h_attn.hip), with the probabilities
// computed again from the operands and the forward's log-sum-exp:
//
//   P_ij = exp(scale q_i.k_j - lse_i)      delta_i = sum_d dout_id out_id
//   dP_ij = dout_i.v_j                     dS_ij = P_ij (dP_ij - delta_i)
//   dv_j = sum_i P_ij dout_i    dq_i = scale sum_j dS_ij k_j    dk_j = scale sum_i dS_ij q_i
//
// One launch for delta, one for the rest: blocks for dk and dv, which keep their
// keys in registers while the queries stream past, and blocks for dq, which keep
// their queries while the keys stream. They compute P and dP twice, seven
// products in place of five, and need no atomic sums, whose order would change
// the result from run to run; side by side they fill the GPU where either alone
// would not (4,096 tokens, 12 heads of 128: 371 -> 355 us; 1,024 tokens, 16 heads of
// 64: 40.5 -> 29.1).
//
// f16: P is rounded as 2^14 P (P is near 1 / keys, below f16's smallest normal
// number from 16,384 keys on), and dS as 2^e dS, e a power of two from the bound
// |dP_ij - delta_i| <= 2 |dout_i| max_j |v_j| that puts the bound just below
// f16's largest number; both factors are taken out of the f32 sums.
#include "t2h_attn_core.h"

namespace t2h {
namespace {

constexpr int kPrepRows = 64;     // rows per block of the first pass, and per entry of the maxima
constexpr float kShiftP = 14.0f;  // f16: P is rounded as 2^kShiftP P

template <typename T> struct HalfRange { static constexpr bool value = false; };
template <> struct HalfRange<_Float16> { static constexpr bool value = true; };

// Largest of the entries of n rows.
__device__ __forceinline__ float largest(const float* entries, int n, int lane) {
    float m = 0.0f;
    for (int t = lane; t * kPrepRows < n; t += 64) m = fmaxf(m, entries[t]);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
    return m;
}
// e with 2^e * 2 sqrt(g2 v2) below 2^16, from the largest squared lengths.
__device__ __forceinline__ float shift_ds(float g2, float v2) {
    const float b = 2.0f * sqrtf(g2) * sqrtf(v2);
    int e = 14 - ((int)((__builtin_bit_cast(uint32_t, b) >> 23) & 255u) - 127);
    e = e > 60 ? 60 : e < -60 ? -60 : e;
    return (float)e;
}

// ---- delta, and row lengths for f16 ---------------------------------------------
// A block takes up to kPrepRows rows of one segment and one head of dout and out
// (or, f16, of v; only keys that count), 16 lanes a row.
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_prep_kernel(AttnBwdArgs a) {
    constexpr int E = D / 16;
    constexpr bool kF16 = HalfRange<T>::value;
    const AttnArgs& f = a.f;
    const int64_t p = block_linear();
    if (p >= a.prep_blocks) return;
    const int u = (int)p;
    const int m = threadIdx.x & 15, rr = threadIdx.x >> 4;
    const int qb = a.prep_q_tiles * f.heads;
    const bool q = u < qb;
    const int per = q ? a.prep_q_tiles : a.prep_k_tiles, w = q ? u : u - qb;
    const int head = w / per;
    int b;
    Rows s = tile_rows<kPrepRows>(q ? f.qs : f.ks, f.nbatch, w - head * per, lane_id(), b);
    if (!q) {
        const int end = segment_keys(f, b).hi;
        s.hi = end < s.hi ? end : s.hi;
    }
    const T* x = q ? static_cast<const T*>(a.dout) + head * a.do_head : static_cast<const T*>(f.v) + head * f.v_head;
    const int64_t stride = q ? a.do_row : f.v_row;
    // all rows' loads first: one wait for memory, not one a row
    constexpr int kR = kPrepRows / 16;
    float most = 0.0f;
    if (s.lo < s.hi) {
        float v[kR][E], o[kR][E], lse[kR];
#pragma unroll
        for (int i = 0; i < kR; ++i) {
            const int at = s.lo + i * 16 + rr, row = at < s.hi ? at : s.hi - 1;
            load_elems<T, E>(x + row * stride + m * E, v[i]);
            if (q) {
                load_elems<T, E>(static_cast<const T*>(f.out) + row * f.o_row + head * f.o_head + m * E, o[i]);
                lse[i] = f.lse[head * f.q_rows + row];
            }
        }
#pragma unroll
        for (int i = 0; i < kR; ++i) {
            const int row = s.lo + i * 16 + rr;
            if (kF16) most = fmaxf(most, row16_sum(sum_sq_all<E>(v[i])));   // (a clamped row's counts anyway)
            if (q) {
                float d = 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) d = fmaf(v[i][e], o[i][e], d);
                d = row16_sum(d);
                if (m == 0 && row < s.hi) {
                    const int64_t at = head * f.q_rows + row;
                    a.delta[at] = d;
                    // a row without keys: P = 0
                    a.lse2[at] = lse[i] == -INFINITY ? INFINITY : lse[i] * kLog2e - (kF16 ? kShiftP : 0.0f);
                }
            }
        }
    }
    if constexpr (kF16) {
        __shared__ float top[16];
        if (m == 0) top[rr] = most;
        __syncthreads();
        if (threadIdx.x == 0) {
#pragma unroll
            for (int i = 1; i < 16; ++i) most = fmaxf(most, top[i]);
            (q ? a.g_most : a.v_most)[w] = most;
        }
    }
}

// ---- dq -------------------------------------------------------------------------
constexpr int kKT = 64;   // keys per tile

template <typename T, int D, int NW, int NT>
__device__ __forceinline__ void dq_block(const AttnBwdArgs& a, uint8_t* lds, int p) {   // lds: k, k, v, v
    using V8 = typename AttnMma<T>::v8;
    constexpr int BQ = NW * NT * 16;
    constexpr int kTile = kKT * D * 2;
    constexpr bool kF16 = HalfRange<T>::value;
    const AttnArgs& f = a.f;
    const int u = xcd_order(p, a.q_blocks);
    const int per_head = f.q_tiles * a.q_split;
    const int head = u / per_head;
    const int rem = u - head * per_head;
    const int split = rem / f.q_tiles;
    int b;
    const Rows qs = tile_rows<BQ>(f.qs, f.nbatch, rem - split * f.q_tiles, lane_id(), b);
    if (qs.lo >= qs.hi) return;
    Rows ks = segment_keys(f, b);
    const int keys = ks.hi - ks.lo;
    if (a.q_split > 1) {
        const int tiles = (ks.hi - ks.lo + kKT - 1) / kKT;
        const int t0 = (int)((int64_t)tiles * split / a.q_split), t1 = (int)((int64_t)tiles * (split + 1) / a.q_split);
        if (t1 < tiles) ks.hi = ks.lo + t1 * kKT;
        ks.lo += t0 * kKT;
    }
    const int n = ks.hi > ks.lo ? (ks.hi - ks.lo + kKT - 1) / kKT : 0;

    const int lane = lane_id(), r = lane & 15, h = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int q0 = qs.lo + wave * (NT * 16);
    const bool active = q0 < qs.hi;
    const int kvh = head / f.group;
    const uint8_t* kb = static_cast<const uint8_t*>(f.k) + kvh * f.k_head * 2;
    const uint8_t* vb = static_cast<const uint8_t*>(f.v) + kvh * f.v_head * 2;
    TileLoad<D, kKT, NW> lk, lv;
    lk.init(wave, lane, f.k_row);
    lv.init(wave, lane, f.v_row);
    const FragAddr<D> fa(lane);
    const float c = f.scale * kLog2e;

    V8 q[NT][D / 32], g[NT][D / 32];
    f32x4 dq[D / 16][NT];
    float l2[NT], de[NT], z[NT], w[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) dq[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        l2[j] = INFINITY;
        de[j] = 0.0f;
        z[j] = 1.0f;
        w[j] = f.scale;
    }
    if (n > 0) {
        lk.issue(kb, ks.lo, ks.hi, lds);
        lv.issue(vb, ks.lo, ks.hi, lds + 2 * kTile);
    }
    if (active && n > 0) {
        float v2 = 0.0f;
        if constexpr (kF16) v2 = largest(a.v_most + kvh * a.prep_k_tiles + first_tile<kPrepRows>(f.ks, b), keys, lane);
        const uint8_t* qb = static_cast<const uint8_t*>(f.q) + (head * f.q_head + (int64_t)q0 * f.q_row) * 2;
        const uint8_t* gb = static_cast<const uint8_t*>(a.dout) + (head * a.do_head + (int64_t)q0 * a.do_row) * 2;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            load_own<T, D>(q[j], qb + 16 * j * f.q_row * 2, qs.hi - q0 - 16 * j, (uint32_t)f.q_row * 2, lane);
            load_own<T, D>(g[j], gb + 16 * j * a.do_row * 2, qs.hi - q0 - 16 * j, (uint32_t)a.do_row * 2, lane);
            const int row = q0 + 16 * j + r;
            if (row < qs.hi) {
                l2[j] = a.lse2[head * f.q_rows + row];
                de[j] = a.delta[head * f.q_rows + row];
            }
            if constexpr (kF16) {
                float g2 = 0.0f;
#pragma unroll
                for (int t = 0; t < D / 32; ++t)
#pragma unroll
                    for (int e = 0; e < 8; ++e) g2 = fmaf((float)g[j][t][e], (float)g[j][t][e], g2);
                g2 += __shfl_xor(g2, 16);
                g2 += __shfl_xor(g2, 32);
                const float e = shift_ds(g2, v2);
                z[j] = exp2_f(e - kShiftP);
                de[j] *= z[j];
                w[j] = f.scale * exp2_f(-e);
            }
        }
    }
    if (n > 0) {
        for (int t = 0; t < n; ++t) {
            const int st = t & 1;
            wait_loads<0>();
            wait_lds_reads();
            tile_barrier();
            if (t + 1 < n) {
                lk.issue(kb, ks.lo + (t + 1) * kKT, ks.hi, lds + (1 - st) * kTile);
                lv.issue(vb, ks.lo + (t + 1) * kKT, ks.hi, lds + (3 - st) * kTile);
            }
            if (!active) continue;
            const int left = ks.hi - ks.lo - t * kKT;
            const uint8_t* kt = lds + st * kTile;
            const uint8_t* vt = lds + (2 + st) * kTile;
#pragma unroll
            for (int s2 = 0; s2 < kKT / 32; ++s2) {
                f32x4 s[2][NT], d[2][NT];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j) s[i][j] = d[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int x = 0; x < D / 32; ++x)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const V8 y = row_frag<T, D>(kt, fa.row, 2 * s2 + i, x);
#pragma unroll
                        for (int j = 0; j < NT; ++j) s[i][j] = AttnMma<T>::run(y, q[j][x], s[i][j]);
                    }
#pragma unroll
                for (int x = 0; x < D / 32; ++x)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const V8 y = row_frag<T, D>(vt, fa.row, 2 * s2 + i, x);
#pragma unroll
                        for (int j = 0; j < NT; ++j) d[i][j] = AttnMma<T>::run(y, g[j][x], d[i][j]);
                    }
                // keys past the last: their score 0 may be far above lse, and P with it beyond any number
                if (left < kKT) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (32 * s2 + 16 * i + 4 * h + e >= left) {
#pragma unroll
                                for (int j = 0; j < NT; ++j) s[i][j][e] = -INFINITY;
                            }
                }
                V8 df[NT];
#pragma unroll
                for (int j = 0; j < NT; ++j) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float pr = exp2_f(fmaf(s[i][j][e], c, -l2[j]));
                            d[i][j][e] = pr * (kF16 ? fmaf(d[i][j][e], z[j], -de[j]) : d[i][j][e] - de[j]);
                        }
                    df[j] = pack_frag<T>(d[0][j], d[1][j]);
                }
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    const V8 x = tr_frag<T, D>(kt, fa.tr, s2, i);
#pragma unroll
                    for (int j = 0; j < NT; ++j) dq[i][j] = AttnMma<T>::run(x, df[j], dq[i][j]);
                }
                if (NT == 1 && a.fine) {
                    const V8 rest = rest_frag<T>(d[0][0], d[1][0], df[0]);
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) dq[i][0] = AttnMma<T>::run(tr_frag<T, D>(kt, fa.tr, s2, i), rest, dq[i][0]);
                }
            }
        }
    }
    if (!active) return;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int row = q0 + 16 * j + r;
        if (row >= qs.hi) continue;
        if (a.q_split > 1) {
            float* po = a.part_q + (((int64_t)split * f.q_rows + row) * f.heads + head) * D + 4 * h;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) *reinterpret_cast<f32x4*>(po + 16 * i) = dq[i][j] * w[j];
        } else {
            T* po = static_cast<T*>(a.dq) + (int64_t)row * a.dq_row + head * a.dq_head + 4 * h;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                typename AttnMma<T>::v4 x;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = (T)(dq[i][j][e] * w[j]);
                *reinterpret_cast<typename AttnMma<T>::v4*>(po + 16 * i) = x;
            }
        }
    }
}

// ---- dk, dv ---------------------------------------------------------------------
constexpr int kQT = 64;   // queries per tile

template <typename T, int D, int NW, int NT>
__device__ __forceinline__ void dkv_block(const AttnBwdArgs& a, uint8_t* lds, int p) {   // lds: q, q, dout, dout, lse2 x 2, delta x 2
    using V8 = typename AttnMma<T>::v8;
    constexpr int BK = NW * NT * 16;
    constexpr int kTile = kQT * D * 2;
    constexpr bool kF16 = HalfRange<T>::value;
    const AttnArgs& f = a.f;
    const int u = xcd_order(p, a.kv_blocks);
    const int per_head = a.k_tiles * a.kv_split;
    const int kvh = u / per_head;
    const int rem = u - kvh * per_head;
    const int split = rem / a.k_tiles;
    int b;
    const Rows ks = tile_rows<BK>(f.ks, f.nbatch, rem - split * a.k_tiles, lane_id(), b);
    if (ks.lo >= ks.hi) return;
    const Rows qs = segment_rows(f.qs, b);
    // keys from k_end on do not count: their gradients are zero
    const Rows seg = segment_keys(f, b);
    const int k_end = seg.hi;

    const int lane = lane_id(), r = lane & 15, h = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int k0 = ks.lo + wave * (NT * 16);
    const bool active = k0 < k_end;
    const int tiles = (qs.hi - qs.lo + kQT - 1) / kQT;
    const int total = ks.lo < k_end ? tiles * f.group : 0;
    const int it0 = (int)((int64_t)total * split / a.kv_split);
    const int it1 = (int)((int64_t)total * (split + 1) / a.kv_split);

    TileLoad<D, kQT, NW> lq, lg;
    lq.init(wave, lane, f.q_row);
    lg.init(wave, lane, a.do_row);
    const FragAddr<D> fa(lane);
    const float c = f.scale * kLog2e;

    V8 k[NT][D / 32], v[NT][D / 32];
    f32x4 dk[D / 16][NT], dv[D / 16][NT];
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) dk[i][j] = dv[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float z = 1.0f, shift = 0.0f;
    if (it0 < it1) {
        if constexpr (kF16) {
            float g2 = 0.0f;
            const int qt0 = first_tile<kPrepRows>(f.qs, b);
            for (int i = 0; i < f.group; ++i)
                g2 = fmaxf(g2, largest(a.g_most + (kvh * f.group + i) * a.prep_q_tiles + qt0, qs.hi - qs.lo, lane));
            const int kt0 = first_tile<kPrepRows>(f.ks, b);
            shift = shift_ds(g2, largest(a.v_most + kvh * a.prep_k_tiles + kt0, seg.hi - seg.lo, lane));
            z = exp2_f(shift - kShiftP);
        }
        // the next tile: query head and first row
        int head = kvh * f.group, row = qs.lo;
        if (it0 > 0) {
            head += it0 / tiles;
            row += it0 % tiles * kQT;
        }
        const auto issue = [&](int st) {
            lq.issue(static_cast<const uint8_t*>(f.q) + head * f.q_head * 2, row, qs.hi, lds + st * kTile);
            lg.issue(static_cast<const uint8_t*>(a.dout) + head * a.do_head * 2, row, qs.hi, lds + (2 + st) * kTile);
            if (wave < 2) {
                const float* src = (wave == 0 ? a.lse2 : a.delta) + (head * f.q_rows + row);
                const int left = qs.hi - row;
                const __amdgpu_buffer_rsrc_t rs = rows_rsrc(reinterpret_cast<const uint8_t*>(src),
                                                            (uint32_t)(left < kQT ? left : kQT) * 4);
                rsrc_to_lds4(rs, lds + 4 * kTile + (2 * wave + st) * kQT * 4, (uint32_t)lane * 4);
            }
            row += kQT;
            if (row >= qs.hi) {
                row = qs.lo;
                ++head;
            }
        };
        const int first = qs.hi - row;
        issue(0);
        if (active) {
            const uint8_t* kb = static_cast<const uint8_t*>(f.k) + (kvh * f.k_head + (int64_t)k0 * f.k_row) * 2;
            const uint8_t* vb = static_cast<const uint8_t*>(f.v) + (kvh * f.v_head + (int64_t)k0 * f.v_row) * 2;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                load_own<T, D>(k[j], kb + 16 * j * f.k_row * 2, k_end - k0 - 16 * j, (uint32_t)f.k_row * 2, lane);
                load_own<T, D>(v[j], vb + 16 * j * f.v_row * 2, k_end - k0 - 16 * j, (uint32_t)f.v_row * 2, lane);
            }
        }
        int left = first;            // of the tile that is worked on: its rows and those of the head's tiles after it
        for (int it = it0; it < it1; ++it) {
            const int st = (it - it0) & 1;
            const int rows = left;
            left = left > kQT ? left - kQT : qs.hi - qs.lo;
            wait_loads<0>();
            wait_lds_reads();
            tile_barrier();
            if (it + 1 < it1) issue(1 - st);
            if (!active) continue;
            const uint8_t* qt = lds + st * kTile;
            const uint8_t* gt = lds + (2 + st) * kTile;
            const float* ls = reinterpret_cast<const float*>(lds + 4 * kTile) + st * kQT;
            const float* de = ls + 2 * kQT;
#pragma unroll 1
            for (int s2 = 0; s2 < kQT / 32 && 32 * s2 < rows; ++s2) {
                f32x4 s[2][NT], d[2][NT];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j) s[i][j] = d[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int t = 0; t < D / 32; ++t)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const V8 x = row_frag<T, D>(qt, fa.row, 2 * s2 + i, t);
#pragma unroll
                        for (int j = 0; j < NT; ++j) s[i][j] = AttnMma<T>::run(x, k[j][t], s[i][j]);
                    }
#pragma unroll
                for (int t = 0; t < D / 32; ++t)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const V8 x = row_frag<T, D>(gt, fa.row, 2 * s2 + i, t);
#pragma unroll
                        for (int j = 0; j < NT; ++j) d[i][j] = AttnMma<T>::run(x, v[j][t], d[i][j]);
                    }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const f32x4 l4 = *reinterpret_cast<const f32x4*>(ls + 32 * s2 + 16 * i + 4 * h);
                    f32x4 d4 = *reinterpret_cast<const f32x4*>(de + 32 * s2 + 16 * i + 4 * h);
                    if (kF16) d4 *= z;
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            s[i][j][e] = exp2_f(fmaf(s[i][j][e], c, -l4[e]));
                            d[i][j][e] = s[i][j][e] * (kF16 ? fmaf(d[i][j][e], z, -d4[e]) : d[i][j][e] - d4[e]);
                        }
                }
                V8 pf[NT], df[NT];
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    pf[j] = pack_frag<T>(s[0][j], s[1][j]);
                    df[j] = pack_frag<T>(d[0][j], d[1][j]);
                }
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    const V8 x = tr_frag<T, D>(gt, fa.tr, s2, i);
#pragma unroll
                    for (int j = 0; j < NT; ++j) dv[i][j] = AttnMma<T>::run(x, pf[j], dv[i][j]);
                }
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    const V8 x = tr_frag<T, D>(qt, fa.tr, s2, i);
#pragma unroll
                    for (int j = 0; j < NT; ++j) dk[i][j] = AttnMma<T>::run(x, df[j], dk[i][j]);
                }
                if (NT == 1 && a.fine) {
                    const V8 pr = rest_frag<T>(s[0][0], s[1][0], pf[0]), dr = rest_frag<T>(d[0][0], d[1][0], df[0]);
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        dv[i][0] = AttnMma<T>::run(tr_frag<T, D>(gt, fa.tr, s2, i), pr, dv[i][0]);
                        dk[i][0] = AttnMma<T>::run(tr_frag<T, D>(qt, fa.tr, s2, i), dr, dk[i][0]);
                    }
                }
            }
        }
    }
    const float wk = f.scale * (kF16 ? exp2_f(-shift) : 1.0f), wv = kF16 ? exp2_f(-kShiftP) : 1.0f;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int row = k0 + 16 * j + r;
        if (row >= ks.hi) continue;
        const bool counts = row < k_end;
        if (a.kv_split > 1) {
            float* pk = a.part_kv + (((int64_t)split * f.k_rows + row) * a.kv_heads + kvh) * D + 4 * h;
            float* pv = pk + (int64_t)a.kv_split * f.k_rows * a.kv_heads * D;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
                *reinterpret_cast<f32x4*>(pk + 16 * i) = counts ? dk[i][j] * wk : zero;
                *reinterpret_cast<f32x4*>(pv + 16 * i) = counts ? dv[i][j] * wv : zero;
            }
        } else {
            T* pk = static_cast<T*>(a.dk) + (int64_t)row * a.dk_row + kvh * a.dk_head + 4 * h;
            T* pv = static_cast<T*>(a.dv) + (int64_t)row * a.dv_row + kvh * a.dv_head + 4 * h;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                typename AttnMma<T>::v4 x, y;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] = counts ? (T)(dk[i][j][e] * wk) : (T)0.0f;
                    y[e] = counts ? (T)(dv[i][j][e] * wv) : (T)0.0f;
                }
                *reinterpret_cast<typename AttnMma<T>::v4*>(pk + 16 * i) = x;
                *reinterpret_cast<typename AttnMma<T>::v4*>(pv + 16 * i) = y;
            }
        }
    }
}

// The side with the longer blocks comes first (q_first), so that the others fill
// the GPU as those end.
template <typename T, int D, int KV, int Q>
__global__ __launch_bounds__(256, 2) void attn_bwd_kernel(AttnBwdArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[4 * kQT * D * 2 + 4 * kQT * 4];
    int64_t p = block_linear();
    if (p >= (int64_t)a.kv_blocks + a.q_blocks) return;
    const int first = a.q_first ? a.q_blocks : a.kv_blocks;
    const bool q = (p < first) == a.q_first;
    if (p >= first) p -= first;
    if (q) dq_block<T, D, 4, Q>(a, lds, (int)p);
    else dkv_block<T, D, 4, KV>(a, lds, (int)p);
}

// Sums of the parts [nsplit, rows, heads, D] in order; blockIdx.z: which of dk,
// dv and dq.
struct SumSet {
    const float* part;
    void* out;
    int64_t row_stride, head_stride, rows;
    const int64_t* offsets;   // rows outside the segments are left alone
    int32_t heads, nsplit;
};
struct SumArgs {
    SumSet set[3];
    int32_t nbatch;
};
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_sum_kernel(SumArgs args) {
    constexpr int E = D / 16;
    const SumSet& a = args.set[blockIdx.z];
    const int64_t u = block_linear() * 16 + threadIdx.x / 16;
    if (u >= a.rows * a.heads) return;
    const int64_t row = u / a.heads;
    const int head = (int)(u - row * a.heads);
    if (a.offsets != nullptr && (row < a.offsets[0] || row >= a.offsets[args.nbatch])) return;
    const int m = threadIdx.x & 15;
    float acc[E] = {};
#pragma unroll 4
    for (int s = 0; s < a.nsplit; ++s) {
        float v[E];
        load_params<E>(a.part + (((int64_t)s * a.rows + row) * a.heads + head) * D + m * E, v);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += v[e];
    }
    store_elems<T, E>(static_cast<T*>(a.out) + row * a.row_stride + head * a.head_stride + m * E, acc);
}

// Four waves a block, two blocks a CU; a wave keeps two 16-token tiles (the large
// form) or one (the small).
constexpr int kRowsLarge = 128, kRowsSmall = 64;   // tokens a block keeps
constexpr int kFine = 64;                          // tokens
constexpr int kSplitRows = 1024;                   // streaming tokens that a part of the large form has at least

// How one side's blocks take their work: the large form, its streaming side in as
// many parts as the GPU's two blocks a CU take at once (dk, dv of 1,029 keys, 12
// heads of 128, the whole pass: 8,192 queries in 2 parts 229 us, 4: 214, 6: 221; 2 x
// 19,902 queries in 2 parts 677 us, 3: 692, 6: 718); where the parts would be too
// short for 1.5 blocks a CU (300 queries, 3,000 keys: large 57.6 us, small 51.5),
// and for segments no longer than its tile (64 of 37 tokens, 16 heads of 64, each
// side's blocks alone: 12.2 and 12.5 us, small 8.5 and 9.9), the small form, in
// parts of 128 streaming tokens at least, from 512 on (64 queries, 1,029 keys, 16
// heads of 64: in parts of 128 15.7 us, 256 16.0, 512 21; 300 queries and keys: 2
// parts 16.6, one 12.1). Two blocks a CU there: 24 us for 20.
// Where both sides' small blocks are fewer than the CUs, the parts are such that
// all blocks of both take one CU each for about as long, 256 tokens at least (512
// queries and keys, 16 heads of 64: each side by itself 2 parts 23.6 us, one 17.1;
// 4 heads of 128, 1,024: 4 parts 36.6, 2 38.7; 512 and 2,000, 2 heads 32.0, 29.0).
// Few queries or few keys (kFine in all): P and dS keep twice the type's bits, as
// two products. Such calls wait for memory, not for the matrix cores, and in their
// results a few terms of a sum weigh most, whose rounding does not average out
// (one query, 10,474 keys, f16: dk is 3.4e-4 off in the 2-norm, and so as little
// as its own rounding, 2.2e-4; 16 queries, 60,000 keys 323 -> 381 us).
struct Plan { bool small; int split; int64_t blocks; };   // blocks: unsplit
Plan plan_of(const AttnSide& kept, int64_t stream, int32_t nbatch, int32_t heads, bool fine) {
    const int64_t cu = device_cu_count(), per = (int64_t)nbatch * heads;
    const int64_t large = ((int64_t)kept.share + kRowsLarge - 1) / kRowsLarge * per;
    const int64_t small = ((int64_t)kept.share + kRowsSmall - 1) / kRowsSmall * per;
    const int64_t most = stream / kSplitRows > 1 ? stream / kSplitRows : 1;
    Plan p{};
    p.small = large * most * 2 < 3 * cu || kept.share <= kRowsSmall || fine;
    int64_t n = 1;
    if (p.small) {
        n = stream < 512 ? 1 : cu / (small > 0 ? small : 1);
        if (n > stream / 128) n = stream / 128;
    } else if (large * 2 < 3 * cu) {
        n = 2 * cu / large;
        if (n > most) n = most;
    }
    p.split = (int)(n < 1 ? 1 : n > 64 ? 64 : n);
    p.blocks = p.small ? small : large;
    return p;
}
// Parts for both sides at once, where both have the same form; a block of dk, dv
// does 4 products a streaming token, one of dq 3. Large blocks that fill the GPU's
// places together stay whole on a side where one is no longer than a place's share
// (2,048 tokens, 16 heads of 64, 512 blocks: each side in 2 parts 88 us, whole 71).
void share_cus(Plan& q, int64_t keys, Plan& kv, int64_t queries) {
    const int64_t cu = device_cu_count(), blocks = q.blocks + kv.blocks;
    const int64_t work = q.blocks * keys * 3 + kv.blocks * queries * 4;
    if (q.small && kv.small && blocks <= cu) {
        const int64_t each = work / (cu * 4), len = each > 256 ? each : 256;
        const auto parts = [len](int64_t stream) {
            const int64_t n = (stream + len / 2) / len;
            return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
        };
        q.split = parts(keys);
        kv.split = parts(queries);
    } else if (!q.small && !kv.small && blocks >= 2 * cu) {
        const int64_t share = work / (2 * cu);
        if (keys * 12 <= share * 5) q.split = 1;
        if (queries * 16 <= share * 5) kv.split = 1;
    }
}

template <typename T, int D, int KV, int Q>
void launch_forms(AttnBwdArgs& a, hipStream_t s) {
    AttnArgs& f = a.f;
    a.k_tiles = (int32_t)tile_count(f.ks, f.nbatch, KV * 64);
    f.q_tiles = (int32_t)tile_count(f.qs, f.nbatch, Q * 64);
    a.kv_blocks = a.k_tiles * a.kv_split * a.kv_heads;
    a.q_blocks = f.q_tiles * a.q_split * f.heads;
    const int64_t blocks = (int64_t)a.kv_blocks + a.q_blocks;
    if (blocks > 0) hipLaunchKernelGGL((attn_bwd_kernel<T, D, KV, Q>), grid_1d(blocks), dim3(256), 0, s, a);
}

template <typename T, int D>
hipError_t launch_d(AttnBwdArgs a, hipStream_t s) {
    const AttnArgs& f = a.f;
    if (a.prep_blocks > 0) hipLaunchKernelGGL((attn_prep_kernel<T, D>), grid_1d(a.prep_blocks), dim3(256), 0, s, a);
    if (a.kv_small) a.q_small ? launch_forms<T, D, 1, 1>(a, s) : launch_forms<T, D, 1, 2>(a, s);
    else a.q_small ? launch_forms<T, D, 2, 1>(a, s) : launch_forms<T, D, 2, 2>(a, s);
    SumArgs m{};
    m.nbatch = f.nbatch;
    int sets = 0;
    int64_t units = 0;
    const auto add = [&](const float* part, void* out, int64_t row, int64_t head, int64_t rows, const AttnSide& side,
                         int32_t heads, int32_t nsplit) {
        m.set[sets++] = SumSet{part, out, row, head, rows, side.offsets, heads, nsplit};
        if (rows * heads > units) units = rows * heads;
    };
    if (a.kv_split > 1 && f.k_rows > 0) {
        const float* pv = a.part_kv + a.kv_split * f.k_rows * a.kv_heads * D;
        add(a.part_kv, a.dk, a.dk_row, a.dk_head, f.k_rows, f.ks, a.kv_heads, a.kv_split);
        add(pv, a.dv, a.dv_row, a.dv_head, f.k_rows, f.ks, a.kv_heads, a.kv_split);
    }
    if (a.q_split > 1 && f.q_rows > 0)
        add(a.part_q, a.dq, a.dq_row, a.dq_head, f.q_rows, f.qs, f.heads, a.q_split);
    if (sets > 0) {
        dim3 grid = grid_1d((units + 15) / 16);
        grid.z = sets;
        hipLaunchKernelGGL((attn_sum_kernel<T, D>), grid, dim3(256), 0, s, m);
    }
    return hipGetLastError();
}

int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

}  // namespace

// The workspace: delta and lse2 [heads, q_rows], the maxima (f16), then the
// parts of whichever of dk, dv and dq are split.
int64_t attn_bwd_plan(AttnBwdArgs& a, void* workspace) {
    AttnArgs& f = a.f;
    a.prep_q_tiles = (int32_t)tile_count(f.qs, f.nbatch, kPrepRows);
    a.prep_k_tiles = (int32_t)tile_count(f.ks, f.nbatch, kPrepRows);
    a.prep_blocks = a.prep_q_tiles * f.heads + (f.dtype == T2H_F16 ? a.prep_k_tiles * a.kv_heads : 0);
    const bool fine = f.q_rows <= kFine || f.k_rows <= kFine;
    const int64_t queries = (int64_t)f.qs.share * f.group;    // that a key's block reads
    Plan q = plan_of(f.qs, f.ks.share, f.nbatch, f.heads, fine);
    Plan kv = plan_of(f.ks, queries, f.nbatch, a.kv_heads, fine);
    share_cus(q, f.ks.share, kv, queries);
    a.q_small = q.small;
    a.q_split = q.split;
    a.kv_small = kv.small;
    a.fine = fine;
    a.kv_split = kv.split;
    // a block's products: streaming tokens x kept tiles a wave x 4 or 3
    a.q_first = (int64_t)f.ks.share / q.split * (q.small ? 1 : 2) * 3 >
                queries / kv.split * (kv.small ? 1 : 2) * 4;
    uint8_t* w = static_cast<uint8_t*>(workspace);
    int64_t at = 0;
    const auto take = [&](int64_t floats) {
        float* p = reinterpret_cast<float*>(w + at);
        at += up256(floats * 4);
        return p;
    };
    a.delta = take(f.q_rows * f.heads);
    a.lse2 = take(f.q_rows * f.heads);
    a.g_most = take((f.q_rows / kPrepRows + f.nbatch) * f.heads);     // as many with offsets as without
    a.v_most = take((f.k_rows / kPrepRows + f.nbatch) * a.kv_heads);
    const int64_t pk = a.kv_split > 1 ? 2 * (int64_t)a.kv_split * f.k_rows * a.kv_heads * f.head_dim : 0;
    const int64_t pq = a.q_split > 1 ? (int64_t)a.q_split * f.q_rows * f.heads * f.head_dim : 0;
    a.part_kv = take(pk);
    a.part_q = take(pq);
    return at;
}

hipError_t launch_attn_bwd(const AttnBwdArgs& a, hipStream_t s) {
    if (a.f.dtype == T2H_F16) return a.f.head_dim == 128 ? launch_d<_Float16, 128>(a, s) : launch_d<_Float16, 64>(a, s);
    return a.f.head_dim == 128 ? launch_d<__bf16, 128>(a, s) : launch_d<__bf16, 64>(a, s);
}

}  // namespace t2h
