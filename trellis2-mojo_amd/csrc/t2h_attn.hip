// Attention over ragged or dense batches on the matrix cores.
//
//   s_ij = scale * sum_d q_id k_jd       lse_i = log sum_j exp(s_ij)
//   out_i = sum_j exp(s_ij - lse_i) v_j
#include "t2h_attn_core.h"

namespace t2h {
namespace {

constexpr int kKT = 64;   // keys per tile

// The scores are kept unscaled; with c = scale * log2(e), p = exp2(c s - mc), mc
// = c * (a reference close to the row's running maximum).
template <typename T, int D, int NW, bool SPLIT>
__global__ __launch_bounds__(NW * 64, 2) void attn_kernel(AttnArgs a) {
    using V8 = typename AttnMma<T>::v8;
    constexpr int BQ = NW * 32;
    constexpr int kTile = kKT * D * 2;
    constexpr float kRise = 8.0f;   // the reference follows the maximum once it is this far above (log2)
    __shared__ __attribute__((aligned(16))) uint8_t lds[4 * kTile];   // K, K, V, V
    const int64_t p = block_linear();
    if (p >= a.nblocks) return;
    const int u = xcd_order((int)p, a.nblocks);
    const int per_head = a.q_tiles * a.nsplit;
    const int head = u / per_head;
    const int rem = u - head * per_head;
    const int split = SPLIT ? rem / a.q_tiles : 0;
    int b;
    const Rows qs = tile_rows<BQ>(a.qs, a.nbatch, rem - split * a.q_tiles, b);
    if (qs.lo >= qs.hi) return;
    Rows ks = segment_keys(a, b);
    if constexpr (SPLIT) {
        const int tiles = (ks.hi - ks.lo + kKT - 1) / kKT;
        const int t0 = (int)((int64_t)tiles * split / a.nsplit), t1 = (int)((int64_t)tiles * (split + 1) / a.nsplit);
        if (t1 < tiles) ks.hi = ks.lo + t1 * kKT;
        ks.lo += t0 * kKT;
    }
    const int n = ks.hi > ks.lo ? (ks.hi - ks.lo + kKT - 1) / kKT : 0;

    const int lane = lane_id(), r = lane & 15, h = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int q0 = qs.lo + wave * 32;
    const bool active = q0 < qs.hi;
    const int kvh = head / a.group;
    const uint8_t* kb = static_cast<const uint8_t*>(a.k) + kvh * a.k_head * 2;
    const uint8_t* vb = static_cast<const uint8_t*>(a.v) + kvh * a.v_head * 2;
    TileLoad<D, kKT, NW> lk, lv;
    lk.init(wave, lane, a.k_row);
    lv.init(wave, lane, a.v_row);
    const FragAddr<D> fa(lane);

    V8 q[2][D / 32];
    f32x4 o[D / 16][2];
    float mc[2] = {0.0f, 0.0f}, thr[2], l[2] = {0.0f, 0.0f};
    thr[0] = thr[1] = -INFINITY;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[i][0] = o[i][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const float c = a.scale * kLog2e;

    if (n > 0) {
        lk.issue(kb, ks.lo, ks.hi, lds);
        if (active) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
                load_own<T, D>(q[j], static_cast<const uint8_t*>(a.q) + head * a.q_head * 2 + (int64_t)(q0 + 16 * j) * a.q_row * 2,
                               qs.hi - q0 - 16 * j, (uint32_t)a.q_row * 2, lane);
        }
        wait_loads<0>();
        tile_barrier();
        lv.issue(vb, ks.lo, ks.hi, lds + 2 * kTile);
        if (n > 1) lk.issue(kb, ks.lo + kKT, ks.hi, lds + kTile);
        f32x4 s[4][2];
        const auto scores = [&](const uint8_t* kt, f32x4 (&x)[4][2]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i][0] = x[i][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int t = 0; t < D / 32; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const V8 f = row_frag<T, D>(kt, fa.row, i, t);
#pragma unroll
                    for (int j = 0; j < 2; ++j) x[i][j] = AttnMma<T>::run(f, q[j][t], x[i][j]);
                }
        };
        // keys from `left` on do not count
        const auto mask = [&](f32x4 (&x)[4][2], int left) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (16 * i + 4 * h + e >= left) x[i][0][e] = x[i][1][e] = -INFINITY;
        };
        const auto follow = [&](const f32x4 (&x)[4][2]) {
            float top[2];
            bool rise = false;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                top[j] = x[0][j][0];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) top[j] = fmaxf(top[j], x[i][j][e]);
                top[j] *= c;
                rise |= top[j] > thr[j];
            }
            if (__any(rise)) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float t = fmaxf(top[j], __shfl_xor(top[j], 16));
                    t = fmaxf(t, __shfl_xor(t, 32));
                    if (t > thr[j]) {
                        const float alpha = thr[j] == -INFINITY ? 0.0f : exp2_f(mc[j] - t);
                        mc[j] = t;
                        thr[j] = t + kRise;
                        l[j] *= alpha;
#pragma unroll
                        for (int i = 0; i < D / 16; ++i) o[i][j] *= alpha;
                    }
                }
            }
        };
        if (active) {
            scores(lds, s);
            if (n == 1) mask(s, ks.hi - ks.lo);
            follow(s);
        }
        for (int t = 0; t < n; ++t) {
            wait_loads<0>();
            wait_lds_reads();
            tile_barrier();
            const int st = t & 1;
            if (t + 1 < n) lv.issue(vb, ks.lo + (t + 1) * kKT, ks.hi, lds + (3 - st) * kTile);
            if (t + 2 < n) lk.issue(kb, ks.lo + (t + 2) * kKT, ks.hi, lds + st * kTile);
            if (!active) continue;
            f32x4 sn[4][2];
            if (t + 1 < n) scores(lds + (1 - st) * kTile, sn);
            V8 pf[2][2];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int k2 = 0; k2 < 2; ++k2) {
#pragma unroll
                    for (int i = 2 * k2; i < 2 * k2 + 2; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            s[i][j][e] = exp2_f(fmaf(s[i][j][e], c, -mc[j]));
                            l[j] += s[i][j][e];
                        }
                    pf[j][k2] = pack_frag<T>(s[2 * k2][j], s[2 * k2 + 1][j]);
                }
            const uint8_t* vt = lds + (2 + st) * kTile;
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    const V8 f = tr_frag<T, D>(vt, fa.tr, k2, i);
#pragma unroll
                    for (int j = 0; j < 2; ++j) o[i][j] = AttnMma<T>::run(f, pf[j][k2], o[i][j]);
                }
            if (t + 1 < n) {
#pragma unroll
                for (int i = 0; i < 4; ++i) s[i][0] = sn[i][0], s[i][1] = sn[i][1];
                if (t + 2 == n) mask(s, ks.hi - ks.lo - (t + 1) * kKT);
                follow(s);
            }
        }
    }
    if (!active) return;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        l[j] += __shfl_xor(l[j], 16);
        l[j] += __shfl_xor(l[j], 32);
        const int row = q0 + 16 * j + r;
        if (row >= qs.hi) continue;
        const float inv = l[j] == 0.0f ? 0.0f : 1.0f / l[j];
        const float lse2 = l[j] == 0.0f ? -INFINITY : mc[j] + __builtin_amdgcn_logf(l[j]);
        if constexpr (SPLIT) {
            if (h == 0) a.part_lse[((int64_t)split * a.heads + head) * a.q_rows + row] = lse2;
            float* po = a.part + (((int64_t)split * a.q_rows + row) * a.heads + head) * D + 4 * h;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) *reinterpret_cast<f32x4*>(po + 16 * i) = o[i][j] * inv;
        } else {
            if (a.lse != nullptr && h == 0) a.lse[head * a.q_rows + row] = lse2 * kLn2;
            T* po = static_cast<T*>(a.out) + (int64_t)row * a.o_row + head * a.o_head + 4 * h;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                typename AttnMma<T>::v4 w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = (T)(o[i][j][e] * inv);
                *reinterpret_cast<typename AttnMma<T>::v4*>(po + 16 * i) = w;
            }
        }
    }
}

// Join of the splits: out = sum_s exp2(lse_s - lse) out_s. One DPP row of 16
// lanes per (row, head), D / 16 elements a lane.
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
    constexpr int E = D / 16;
    const int64_t u = block_linear() * 16 + threadIdx.x / 16;
    if (u >= a.q_rows * a.heads) return;
    const int64_t row = u / a.heads;
    const int head = (int)(u - row * a.heads);
    const int m = threadIdx.x & 15;
    if (a.qs.offsets != nullptr && (row < a.qs.offsets[0] || row >= a.qs.offsets[a.nbatch])) return;
    float top = -INFINITY;
    for (int s = 0; s < a.nsplit; ++s) top = fmaxf(top, a.part_lse[((int64_t)s * a.heads + head) * a.q_rows + row]);
    float acc[E] = {}, sum = 0.0f;
    for (int s = 0; s < a.nsplit; ++s) {
        const float l = a.part_lse[((int64_t)s * a.heads + head) * a.q_rows + row];
        const float w = l == -INFINITY ? 0.0f : exp2_f(l - top);
        float v[E];
        load_params<E>(a.part + (((int64_t)s * a.q_rows + row) * a.heads + head) * D + m * E, v);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(w, v[e], acc[e]);
        sum += w;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= inv;
    store_elems<T, E>(static_cast<T*>(a.out) + (int64_t)row * a.o_row + head * a.o_head + m * E, acc);
    if (a.lse != nullptr && m == 0)
        a.lse[head * a.q_rows + row] = sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

constexpr int kWaves = 8;

template <typename T, int D>
hipError_t launch_d(AttnArgs a, hipStream_t s) {
    a.q_tiles = (int32_t)tile_count(a.qs, a.nbatch, kWaves * 32);
    a.nblocks = a.q_tiles * a.nsplit * a.heads;
    if (a.nsplit > 1) {
        hipLaunchKernelGGL((attn_kernel<T, D, kWaves, true>), grid_1d(a.nblocks), dim3(kWaves * 64), 0, s, a);
        const int64_t nb = (a.q_rows * a.heads + 15) / 16;
        hipLaunchKernelGGL((attn_join_kernel<T, D>), grid_1d(nb), dim3(256), 0, s, a);
    } else {
        hipLaunchKernelGGL((attn_kernel<T, D, kWaves, false>), grid_1d(a.nblocks), dim3(kWaves * 64), 0, s, a);
    }
    return hipGetLastError();
}

}  // namespace

int attn_splits(const AttnArgs& a) {
    const int64_t tiles = tile_count(a.qs, a.nbatch, kWaves * 32) * a.heads;
    const int64_t cu = device_cu_count();
    const int64_t keys = a.k_rows / a.nbatch;
    int64_t n = cu / (tiles > 0 ? tiles : 1);
    if (n > keys / 128) n = keys / 128;
    if (n > 64) n = 64;
    return n < 1 ? 1 : (int)n;
}

int64_t attn_split_bytes(const AttnArgs& a, int nsplit) {
    return nsplit < 2 ? 0 : (int64_t)nsplit * a.q_rows * a.heads * (a.head_dim + 1) * 4;
}

hipError_t launch_attn(AttnArgs a, hipStream_t s) {
    if (a.dtype == T2H_F16) return a.head_dim == 128 ? launch_d<_Float16, 128>(a, s) : launch_d<_Float16, 64>(a, s);
    return a.head_dim == 128 ? launch_d<__bf16, 128>(a, s) : launch_d<__bf16, 64>(a, s);
}

}  // namespace t2h
