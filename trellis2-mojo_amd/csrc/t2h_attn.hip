// Attention over ragged or dense batches on the matrix cores.
//
//   s_ij = scale * sum_d q_id k_jd       lse_i = log sum_j exp(s_ij)
//   out_i = sum_j exp(s_ij - lse_i) v_j
//
// One pass over the keys with each row's running sum of exponentials and a
// reference m near its running maximum: out = sum_j exp(s_ij - m) v_j / sum_j
// exp(s_ij - m) for any m. m moves only when a tile's maximum is more than 2^8
// above it, so most tiles rescale nothing, and the exponentials stay below 2^8 (f16
// holds 2^16).
//
// 4 D operations a score on the matrix cores, one exponential: from some hundred
// queries on the products bound it. There the tiles and their order serve to keep
// the matrix cores fed: the next tile's scores run under this tile's exponentials,
// K and V come to LDS one tile ahead, their fragments serve 32 queries, and two
// blocks a CU cover each other's barriers. Measured (f16, 12 heads of 128): two
// segments of 39,804 tokens in all 4.33 ms, 1,130 TFLOP/s, where the library's
// largest products reach 1,300 on the same card; the matrix cores are busy 57 % of
// the cycles, LDS has no conflicts, and the clock falls to 1.7-2.0 GHz of 2.4: power
// bounds both. 4,096 tokens (bf16) 110 us, 935 TFLOP/s: 384 blocks on 512 places.
// Few queries read K and V once from memory: 100,000 keys 118 us, 5.2 TB/s.
#include <type_traits>

#include "t2h_attn_core.h"

namespace t2h {
namespace {

// A block takes BQ = NW * NT * 16 queries of one head; wave w of the NW * KG
// keeps NT * 16 of them in registers, as B operands, with the output that its
// share of the keys gives: of every KG * KT keys that come to LDS (two slots)
// group w / NW takes KT. The groups' outputs are joined in LDS at the end.
// The scores are kept unscaled; with c = scale * log2(e), p = exp2(c s - mc), mc
// = c * (a reference close to the row's running maximum).
template <typename T, int D, int NW, int NT, int KT, int KG, bool SPLIT>
__global__ __launch_bounds__(NW * KG * 64, 2) void attn_kernel(AttnArgs a) {
    using V8 = typename AttnMma<T>::v8;
    constexpr int BQ = NW * NT * 16, BK = KG * KT, kS = KT / 16, kP = KT / 32;
    constexpr int kTile = KT * D * 2, kStage = KG * kTile;
    // Few queries wait for memory, not for the matrix cores: there the
    // probabilities keep twice the type's bits, as two products.
    constexpr bool FINE = KG > 1;
    constexpr float kRise = 8.0f;   // the reference follows the maximum once it is this far above (log2)
    __shared__ __attribute__((aligned(16))) uint8_t lds[4 * kStage];   // K, K, V, V
    const int64_t p = block_linear();
    if (p >= a.nblocks) return;
    const int lane = lane_id(), r = lane & 15, h = lane >> 4;
    const int u = xcd_order((int)p, a.nblocks);
    const int per_head = a.q_tiles * a.nsplit;
    const int head = u / per_head;
    const int rem = u - head * per_head;
    const int split = SPLIT ? rem / a.q_tiles : 0;
    int b;
    const Rows qs = tile_rows<BQ>(a.qs, a.nbatch, rem - split * a.q_tiles, lane, b);
    if (qs.lo >= qs.hi) return;
    Rows ks = segment_keys(a, b);
    if constexpr (SPLIT) {
        const int tiles = (ks.hi - ks.lo + KT - 1) / KT;
        const int t0 = (int)((int64_t)tiles * split / a.nsplit), t1 = (int)((int64_t)tiles * (split + 1) / a.nsplit);
        if (t1 < tiles) ks.hi = ks.lo + t1 * KT;
        ks.lo += t0 * KT;
    }
    const int n = ks.hi > ks.lo ? (ks.hi - ks.lo + BK - 1) / BK : 0;

    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int qw = KG == 1 ? wave : wave % NW, kg = KG == 1 ? 0 : wave / NW;
    const int q0 = qs.lo + qw * (NT * 16);
    const bool active = q0 < qs.hi;
    const int kvh = head / a.group;
    const uint8_t* kb = static_cast<const uint8_t*>(a.k) + kvh * a.k_head * 2;
    const uint8_t* vb = static_cast<const uint8_t*>(a.v) + kvh * a.v_head * 2;
    TileLoad<D, BK, NW * KG> lk, lv;
    lk.init(wave, lane, a.k_row);
    lv.init(wave, lane, a.v_row);
    const FragAddr<D> fa(lane);

    V8 q[NT][D / 32];
    f32x4 o[D / 16][NT];
    float mc[NT], thr[NT], l[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        mc[j] = l[j] = 0.0f;
        thr[j] = -INFINITY;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const float c = a.scale * kLog2e;

    if (n > 0) {
        // q and the first tiles; K's second is fetched as zeros where there is none
        if (active) {
#pragma unroll
            for (int j = 0; j < NT; ++j)
                load_own<T, D>(q[j], static_cast<const uint8_t*>(a.q) + head * a.q_head * 2 + (int64_t)(q0 + 16 * j) * a.q_row * 2,
                               qs.hi - q0 - 16 * j, (uint32_t)a.q_row * 2, lane);
        }
        lk.issue(kb, ks.lo, ks.hi, lds);
        lv.issue(vb, ks.lo, ks.hi, lds + 2 * kStage);
        lk.issue(kb, ks.lo + BK, ks.hi, lds + kStage);
        wait_loads<2 * decltype(lk)::kLoads>();
        tile_barrier();
        f32x4 sa[kS][NT], sb[kS][NT];
        const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
        const auto scores = [&](const uint8_t* kt, f32x4 (&x)[kS][NT]) {
#pragma unroll
            for (int i = 0; i < kS; ++i)
#pragma unroll
                for (int t = 0; t < D / 32; ++t) {
                    const V8 f = row_frag<T, D>(kt, fa.row, i, t);
#pragma unroll
                    for (int j = 0; j < NT; ++j) x[i][j] = AttnMma<T>::run(f, q[j][t], t == 0 ? zero : x[i][j]);
                }
        };
        // keys from `left` on do not count
        const auto mask = [&](f32x4 (&x)[kS][NT], int left) {
#pragma unroll
            for (int i = 0; i < kS; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (16 * i + 4 * h + e >= left) {
#pragma unroll
                        for (int j = 0; j < NT; ++j) x[i][j][e] = -INFINITY;
                    }
        };
        const auto tops = [&](const f32x4 (&x)[kS][NT], float (&top)[NT]) {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                top[j] = x[0][j][0];
#pragma unroll
                for (int i = 0; i < kS; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) top[j] = fmaxf(top[j], x[i][j][e]);
            }
        };
        const auto follow = [&](float (&top)[NT]) {
            bool rise = false;
#pragma unroll
            for (int j = 0; j < NT; ++j) rise |= top[j] * c > thr[j];
            if (__any(rise)) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    float t = fmaxf(top[j], __shfl_xor(top[j], 16));
                    t = fmaxf(t, __shfl_xor(t, 32)) * c;
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
        float top[NT];
        const int mine = ks.hi - ks.lo - kg * KT;      // keys from the group's first on
        if (active) {
            scores(lds + kg * kTile, sa);
            if (mine < KT) mask(sa, mine);
            tops(sa, top);
            follow(top);
        }
        // Tile t: its probabilities from s while the matrix cores make the next
        // tile's scores (MORE), then its part of the output.
        const auto tile = [&](auto more, int t, f32x4 (&s)[kS][NT], f32x4 (&sn)[kS][NT]) {
            constexpr bool MORE = decltype(more)::value;
            wait_loads<0>();
            wait_lds_reads();
            tile_barrier();
            const int st = t & 1;
            if (MORE) lv.issue(vb, ks.lo + (t + 1) * BK, ks.hi, lds + (3 - st) * kStage);
            if (t + 2 < n) lk.issue(kb, ks.lo + (t + 2) * BK, ks.hi, lds + st * kStage);
            if (!active) return;
            if (MORE) scores(lds + (1 - st) * kStage + kg * kTile, sn);
            V8 pf[NT][kP];
#pragma unroll
            for (int k2 = 0; k2 < kP; ++k2)
#pragma unroll
                for (int j = 0; j < NT; ++j) {
#pragma unroll
                    for (int i = 2 * k2; i < 2 * k2 + 2; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            s[i][j][e] = exp2_f(fmaf(s[i][j][e], c, -mc[j]));
                            l[j] += s[i][j][e];
                        }
                    pf[j][k2] = pack_frag<T>(s[2 * k2][j], s[2 * k2 + 1][j]);
                }
            const uint8_t* vt = lds + (2 + st) * kStage + kg * kTile;
#pragma unroll
            for (int k2 = 0; k2 < kP; ++k2)
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    const V8 f = tr_frag<T, D>(vt, fa.tr, k2, i);
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        o[i][j] = AttnMma<T>::run(f, pf[j][k2], o[i][j]);
                        if constexpr (FINE) o[i][j] = AttnMma<T>::run(f, rest_frag<T>(s[2 * k2][j], s[2 * k2 + 1][j], pf[j][k2]), o[i][j]);
                    }
                }
            if (MORE) {
                tops(sn, top);
                const int left = mine - (t + 1) * BK;
                if (left < KT) {
                    mask(sn, left);
                    tops(sn, top);
                }
                follow(top);
            }
        };
        constexpr std::true_type more{};
        constexpr std::false_type last{};
        int t = 0;
        for (; t + 2 < n; t += 2) {
            tile(more, t, sa, sb);
            tile(more, t + 1, sb, sa);
        }
        if (t + 1 < n) {
            tile(more, t, sa, sb);
            tile(last, t + 1, sb, sa);
        } else {
            tile(last, t, sa, sb);
        }
    }
    if constexpr (KG > 1) {
        // join of the groups: reference, sum and output of groups 1.. through LDS
        constexpr int kFrags = D / 16 * NT;
        static_assert((KG - 1) * NW * (kFrags * 16 + NT * 12) * 64 <= 4 * kStage, "the join fits the tiles' LDS");
        f32x4* po = reinterpret_cast<f32x4*>(lds);
        float* pm = reinterpret_cast<float*>(lds + (KG - 1) * NW * kFrags * 1024);
        wait_lds_reads();
        tile_barrier();
        if (kg > 0) {
            const int at = wave - NW;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
#pragma unroll
                for (int i = 0; i < D / 16; ++i) po[(at * kFrags + i * NT + j) * 64 + lane] = o[i][j];
                float* m = pm + ((at * NT + j) * 64 + lane) * 3;
                m[0] = mc[j];
                m[1] = thr[j];
                m[2] = l[j];
            }
        }
        wait_lds_reads();
        tile_barrier();
        if (kg > 0) return;
#pragma unroll
        for (int g = 1; g < KG; ++g) {
            const int at = (g - 1) * NW + qw;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const float* m = pm + ((at * NT + j) * 64 + lane) * 3;
                const float m1 = m[0], t1 = m[1], l1 = m[2];
                if (t1 == -INFINITY && l1 == 0.0f) continue;      // a group without keys (its sum is NaN where its scores are)
                const float top = thr[j] == -INFINITY ? m1 : fmaxf(mc[j], m1);
                const float w0 = thr[j] == -INFINITY ? 0.0f : exp2_f(mc[j] - top), w1 = exp2_f(m1 - top);
                mc[j] = top;
                thr[j] = t1;
                l[j] = fmaf(l[j], w0, l1 * w1);
#pragma unroll
                for (int i = 0; i < D / 16; ++i) o[i][j] = o[i][j] * w0 + po[(at * kFrags + i * NT + j) * 64 + lane] * w1;
            }
        }
    }
    if (!active) return;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
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

// Join of the splits: out = sum_s exp2(lse_s - lse) out_s. 16 lanes take a (row,
// head), D / 16 elements a lane, and its splits in turn; MANY: a block's 16 such
// strands share the splits of one (row, head), and meet in LDS. Up to 8 splits (many
// rows) one strand each; more would be a chain of as many loads (whole calls: 1,000
// queries in 4 splits one strand 17.0 us, 16 20.3; one query in 16 splits 13.2 and
// 9.6, in 64 42 and 24).
template <typename T, int D, bool MANY>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
    constexpr int E = D / 16, kWaves = 4;
    const int wave = threadIdx.x >> 6, lane = lane_id(), m = lane & 15, h = lane >> 4;
    const int64_t total = a.q_rows * a.heads;
    const int strand = wave * 4 + h, first = MANY ? strand : 0;
    const int64_t u0 = MANY ? block_linear() : block_linear() * 16 + strand;
    const int64_t u = u0 < total ? u0 : total - 1;
    const int64_t row = u / a.heads;
    const int head = (int)(u - row * a.heads);
    const float* pl = a.part_lse + head * a.q_rows + row;
    const float* po = a.part + (row * a.heads + head) * D + m * E;
    const int64_t ls = a.heads * a.q_rows, os = ls * D;
    float top = -INFINITY, sum = 0.0f, acc[E] = {};
#pragma unroll 4
    for (int s = first; s < a.nsplit; s += MANY ? 16 : 1) {
        const float l = pl[s * ls];
        float v[E];
        load_params<E>(po + s * os, v);
        const float t = fmaxf(top, l);
        const float w0 = top == -INFINITY ? 0.0f : exp2_f(top - t), w1 = l == -INFINITY ? 0.0f : exp2_f(l - t);
        top = t;
        sum = fmaf(sum, w0, w1);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = acc[e] * w0 + v[e] * w1;
    }
    const auto join = [&](float t1, float s1, const float (&v)[E]) {
        const float t = fmaxf(top, t1);
        const float w0 = top == -INFINITY ? 0.0f : exp2_f(top - t), w1 = t1 == -INFINITY ? 0.0f : exp2_f(t1 - t);
        top = t;
        sum = sum * w0 + s1 * w1;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = acc[e] * w0 + v[e] * w1;
    };
    if constexpr (MANY) {
#pragma unroll
        for (int x = 16; x < 64; x <<= 1) {
            const float t1 = __shfl_xor(top, x), s1 = __shfl_xor(sum, x);
            float v[E];
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = __shfl_xor(acc[e], x);
            join(t1, s1, v);
        }
        __shared__ float lt[kWaves][16], lm[kWaves][16], lo[kWaves][16][E];
        if (h == 0) {
            lt[wave][m] = top;
            lm[wave][m] = sum;
#pragma unroll
            for (int e = 0; e < E; ++e) lo[wave][m][e] = acc[e];
        }
        __syncthreads();
        if (wave > 0) return;
        for (int w = 1; w < kWaves; ++w) {
            float v[E];
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = lo[w][m][e];
            join(lt[w][m], lm[w][m], v);
        }
    }
    if (u0 >= total || (MANY && h > 0)) return;
    if (a.qs.offsets != nullptr && (row < a.qs.offsets[0] || row >= a.qs.offsets[a.nbatch])) return;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= inv;
    store_elems<T, E>(static_cast<T*>(a.out) + row * a.o_row + head * a.o_head + m * E, acc);
    if (a.lse != nullptr && m == 0)
        a.lse[head * a.q_rows + row] = sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

// The kernel's forms: waves, 16-query tiles a wave, keys of a wave's tile, key
// groups.
struct Large { static constexpr int nw = 4, nt = 2, kt = 64; template <int D> static constexpr int kg = 1; };
struct Small { static constexpr int nw = 4, nt = 1, kt = 64; template <int D> static constexpr int kg = 1; };
struct Few { static constexpr int nw = 1, nt = 1, kt = 32; template <int D> static constexpr int kg = D == 64 ? 8 : 4; };
enum Form { kLarge, kSmall, kFew };

// Few: segments of no more queries than its tile, whose other forms' waves would
// be idle (1 query, 16 heads of 64, 512 keys: 6.0 us, small in parts 7.1; 100,000
// keys, 12 heads of 128: 118 and 120); 17 to 48 queries leave it two and three
// tiles that read the keys again (32 queries, 10,474 keys: 21.0, small 18.0).
// Large: where its blocks fill 1.5 places a CU; below, the small form's twice as
// many blocks do better (2,368 queries, 1,029 keys, 16 heads of 64: small 23.6 us,
// large 26.9; 8,192 queries, 12 heads of 128: 73 and 62), and for segments within
// its tile (64 of 37 tokens: 6.9 and 9.5). With heads of 64 a CU holds four small
// blocks, and its time goes by their number: a small block counts 5, a large one 9
// (4,096 tokens: 12 heads, 3 small or 2 large, 66.3 and 74.6 us; 16, 4 or 2, 85.8 and
// 79.1; 20, 5 or 3, 108 and 115; 24, 6 or 3, 126 and 117). With heads of 128 it holds
// two of either (12 heads 120 and 113).

Form form_of(const AttnArgs& a) {
    const int64_t rows = (a.q_rows + a.nbatch - 1) / a.nbatch, cu = device_cu_count();
    if (rows <= 16) return kFew;
    const int64_t per = (int64_t)a.nbatch * a.heads, large = (rows + 127) / 128 * per;
    if (large * 2 < cu * 3 || rows <= 64) return kSmall;
    const auto each = [cu](int64_t blocks) { return (blocks + cu - 1) / cu; };   // blocks on the fullest CU
    if (a.head_dim == 64 && each((rows + 63) / 64 * per) * 5 < each(large) * 9) return kSmall;
    return kLarge;
}

template <typename T, int D, typename F, bool SPLIT>
void launch_form(AttnArgs& a, hipStream_t s) {
    a.q_tiles = (int32_t)tile_count(a.qs, a.nbatch, F::nw * F::nt * 16);
    a.nblocks = a.q_tiles * a.nsplit * a.heads;
    constexpr int kg = F::template kg<D>;
    hipLaunchKernelGGL((attn_kernel<T, D, F::nw, F::nt, F::kt, kg, SPLIT>), grid_1d(a.nblocks), dim3(F::nw * kg * 64), 0, s, a);
}

template <typename T, int D>
hipError_t launch_d(AttnArgs a, hipStream_t s) {
    switch (form_of(a)) {
        case kLarge: launch_form<T, D, Large, false>(a, s); break;
        case kSmall: a.nsplit > 1 ? launch_form<T, D, Small, true>(a, s) : launch_form<T, D, Small, false>(a, s); break;
        default: a.nsplit > 1 ? launch_form<T, D, Few, true>(a, s) : launch_form<T, D, Few, false>(a, s);
    }
    if (a.nsplit > 1) {
        const int64_t units = a.q_rows * a.heads;
        if (a.nsplit > 8) hipLaunchKernelGGL((attn_join_kernel<T, D, true>), grid_1d(units), dim3(256), 0, s, a);
        else hipLaunchKernelGGL((attn_join_kernel<T, D, false>), grid_1d((units + 15) / 16), dim3(256), 0, s, a);
    }
    return hipGetLastError();
}

}  // namespace

// Parts of the keys: as many as idle CUs take, of 128 keys at least. One query,
// replayed, in one part / in parts: 16 heads of 64, 512 keys 6.0 / 7.3 us, 1,029
// keys 8.3 / 8.0 (and a second launch's 2.5 us where the host waits for it); 12
// heads of 128, 1,500 keys 14.7 / 9, 2,058 keys 20 / 9.5, 10,474 keys 92 / 17.7. Parts of
// 1,024 keys at least: 14.6 and 20.3; two blocks a CU: 9.5 and 20.9. 48 queries,
// 1,029 keys 11.2 / 8.3; 300 queries, 10,474 keys 123 / 39.
int attn_splits(const AttnArgs& a) {
    // few queries: keys that a block takes in six turns stay in one launch
    const int64_t one_part = 6 * Few::kt * (a.head_dim == 64 ? Few::kg<64> : Few::kg<128>);
    const int64_t rows = (a.q_rows + a.nbatch - 1) / a.nbatch, keys = a.k_rows / a.nbatch;
    const Form f = form_of(a);
    if (f == kLarge || (f == kFew && keys <= one_part)) return 1;
    const int64_t tiles = (rows + (f == kFew ? 15 : 63)) / (f == kFew ? 16 : 64) * a.nbatch * a.heads;
    int64_t n = device_cu_count() / (tiles > 0 ? tiles : 1);
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
