// Backward pass of the q/k epilogue (t2h_qk.hip): bias, per-head RMS norm and
// rotation, y = R(x / n * gamma * scale) with x = in + bias, n = max(|x|,
// 1e-12), scale = sqrt(head_dim). With dy the gradient of y:
//
//   g  = R^T dy                      (the rotation by the negative angle)
//   w  = g * gamma * scale           xh = x / n
//   dx = (w - xh (xh . w)) / n       (n at its floor, a constant: dx = w / n)
//   dgamma = scale sum_r g * xh      dbias = sum_r dx
//
// and dx = g without a norm. One pass: a wave takes whole rows, several in
// turn, and keeps its lanes' sums of dgamma and dbias in f32 registers; a
// block joins its waves' in LDS and writes one partial row, and a second
// launch sums the partial rows in their order.
//
// Memory bounds it: x, dy and dx once each. The next row's pieces are loaded while
// this one is worked on, and the parameters wait in LDS, not in registers, so that
// three waves fit a SIMD (two for f32 rows): 201,436 tokens, 12 heads of 128, q and
// k (f16) 903 -> 683 us, 5.4 TB/s, more than a large copy's 5.1; 4,096 tokens (f32)
// 50 -> 35 us.
//
// Reference (the forward): sparse/attention/modules.mojo:37-102,
// sparse/attention/rope.mojo:76-134, gpu/attention.mojo:507-563.
#include "t2h_device.h"
#include "t2h_attn.h"
#include "t2h_rope.h"

namespace t2h {
namespace {

constexpr int kW = 4;        // waves per block
constexpr int kShortW = 16;  // ... of the form for few rows
constexpr int kShort = 48;   // rows that it takes

template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
    if constexpr (LPH == 16) return row16_sum(v);
    else return row8_sum(v);
}

// One row's pieces of a wave, as loaded: the next row's are in flight while this
// one is worked on.
template <typename T, int D, int NG, int LPH, bool CACHED> struct RowPieces {
    using L = HeadLanes<T, D, LPH>;
    static constexpr int HPI = 64 / LPH;
    static constexpr int kWords = L::VE * (int)sizeof(T) / 4;   // 4, or 2 (f32 of head_dim 64 has 4 too)
    typedef uint32_t W __attribute__((ext_vector_type(kWords)));
    W w[NG][L::NC];
    __device__ __forceinline__ void load(const T* row, int H, int g, int m) {
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int hh = HPI * i + g < H ? HPI * i + g : H - 1;
#pragma unroll
            for (int j = 0; j < L::NC; ++j) {
                const W* p = reinterpret_cast<const W*>(row + (int64_t)hh * D + L::piece(m, j));
                w[i][j] = CACHED ? *p : __builtin_nontemporal_load(p);
            }
        }
    }
    __device__ __forceinline__ void get(int i, float* f) const {
#pragma unroll
        for (int j = 0; j < L::NC; ++j)
#pragma unroll
            for (int c = 0; c < kWords; ++c) Word<T>::unpack(w[i][j][c], f + j * L::VE + c * Word<T>::N);
    }
};

// Head layout as the forward's (HeadLanes): LPH lanes per head, NG groups of
// 64 / LPH heads. SHORT (few rows): a block takes all rows of one group of heads
// and writes the sums themselves, without a second launch. CACHED: row loads by
// the default policy.
template <typename T, int D, int NG, int W, bool SHORT, bool CACHED>
__global__ __launch_bounds__(W * 64, SHORT ? 4 : sizeof(T) == 2 && NG < 4 ? 3 : 2) void qk_bwd_kernel(QkBwdArgs a, RopeSlots tab) {
    constexpr int LPH = (sizeof(T) == 2 && D == 64) ? 8 : 16;
    constexpr int HPI = 64 / LPH;
    using L = HeadLanes<T, D, LPH>;
    using Pieces = RowPieces<T, D, NG, LPH, CACHED>;
    constexpr int E = L::E, P = L::P, HALF = D / 2;
    // gamma * scale and bias while rows are worked on, the waves' sums afterwards
    __shared__ __attribute__((aligned(16))) float lds[W][NG * HPI * D];
    const int lane = lane_id(), g = lane / LPH, m = lane % LPH;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int which = (int)(blockIdx.x % a.tensors);
    const QkBwdTensor& t = a.t[which];
    const int64_t blk = SHORT ? 0 : blockIdx.x / a.tensors;
    // the block's heads: all, or HPI from head0 on
    const int head0 = SHORT ? (int)(blockIdx.x / a.tensors) * HPI : 0, at0 = head0 * D;
    const int H = SHORT ? (a.heads - head0 < HPI ? a.heads - head0 : HPI) : a.heads, HD = H * D;
    const T* __restrict__ x = static_cast<const T*>(t.x) + at0;
    const T* __restrict__ dy = static_cast<const T*>(t.dy) + at0;
    T* __restrict__ dx = static_cast<T*>(t.dx) + at0;
    const bool norm = t.gamma != nullptr, biased = norm && t.bias != nullptr;
    const bool turn = a.use_rope && a.phases == nullptr;
    const PosSource src{a.coords, a.coord_cols, a.grid_res, a.pos_dim};
    const int my_slot = lane % HALF;
    const int my_axis = turn ? slot_axis(my_slot, a.freq_dim, a.pos_dim) : -1;
    const float my_freq = tab.freq[my_slot];
    const int64_t step = SHORT ? W : a.blocks * W;

    int64_t r = blk * W + wave;
    Pieces xn, gn;
    int pos = 0;
    if (r < a.rows) {
        if (my_axis >= 0) pos = src.at(r, my_axis);
        gn.load(dy + r * a.dy_stride, H, g, m);
        if (norm) xn.load(x + r * a.x_stride, H, g, m);
    }
    if (norm)
        for (int c = threadIdx.x; c < HD; c += W * 64) {
            lds[0][c] = t.gamma[at0 + c] * a.rms_scale;
            if (biased) lds[1][c] = t.bias[at0 + c];
        }
    __syncthreads();
    float sg[NG][E], sb[NG][E];
#pragma unroll
    for (int i = 0; i < NG; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) sg[i][e] = sb[i][e] = 0.0f;
    for (; r < a.rows; r += step) {
        const Pieces xr = xn, gr = gn;
        const int at = pos;
        if (r + step < a.rows) {
            if (my_axis >= 0) pos = src.at(r + step, my_axis);
            gn.load(dy + (r + step) * a.dy_stride, H, g, m);
            if (norm) xn.load(x + (r + step) * a.x_stride, H, g, m);
        }
        float pc[P], ps[P];
        if (turn) {
            float c = 1.0f, s = 0.0f;
            if (my_axis >= 0) sincosf(mul_rn((float)at, my_freq), &s, &c);
#pragma unroll
            for (int p = 0; p < P; ++p) {
                pc[p] = lane_bcast(c, L::slot(m, p));
                ps[p] = lane_bcast(s, L::slot(m, p));
            }
        } else if (a.use_rope) {
            L::phases(a.phases + r % a.phase_rows * (HALF * 2), m, pc, ps);
        }
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const bool valid = HPI * i + g < H;
            const int hl = valid ? HPI * i + g : H - 1;
            float gv[E];
            gr.get(i, gv);
            if (a.use_rope) {
#pragma unroll
                for (int p = 0; p < P; ++p) rotate_pair(gv[2 * p], gv[2 * p + 1], pc[p], -ps[p]);
            }
            if (norm) {
                float xv[E], gm[E];
                xr.get(i, xv);
                if (biased) {
                    float bs[E];
                    L::params(&lds[1][hl * D], m, bs);
#pragma unroll
                    for (int e = 0; e < E; ++e) xv[e] = add_rn(xv[e], bs[e]);
                }
                L::params(&lds[0][hl * D], m, gm);
                float ss = 0.0f, dot = 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) ss = fmaf(xv[e], xv[e], ss);
                ss = head_sum<LPH>(ss);
                const bool floor = ss < 1e-24f;
                const float rn = floor ? 1e12f : __builtin_amdgcn_rsqf(ss);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    xv[e] *= rn;
                    sg[i][e] = fmaf(gv[e], xv[e], sg[i][e]);
                    gv[e] *= gm[e];
                    dot = fmaf(gv[e], xv[e], dot);
                }
                dot = floor ? 0.0f : head_sum<LPH>(dot);
#pragma unroll
                for (int e = 0; e < E; ++e) gv[e] = fmaf(-xv[e], dot, gv[e]) * rn;
            }
#pragma unroll
            for (int e = 0; e < E; ++e) sb[i][e] += gv[e];
            if (valid) L::store(dx + r * a.dx_stride + (int64_t)hl * D, m, gv);
        }
    }
    __syncthreads();
    // the waves' sums joined: dgamma, then dbias
    float* part = a.part + ((int64_t)which * a.blocks + blk) * 2 * HD;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        float* sum = k == 0 ? t.dgamma : t.dbias;
        if (sum == nullptr) continue;
#pragma unroll
        for (int i = 0; i < NG; ++i)
            if (HPI * i + g < H) {
#pragma unroll
                for (int e = 0; e < E; ++e) lds[wave][(HPI * i + g) * D + L::elem(m, e)] = k == 0 ? sg[i][e] : sb[i][e];
            }
        __syncthreads();
        for (int c = threadIdx.x; c < HD; c += W * 64) {
            float s = lds[0][c];
#pragma unroll
            for (int w = 1; w < W; ++w) s += lds[w][c];
            if constexpr (SHORT) sum[at0 + c] = k == 0 ? s * a.rms_scale : s;
            else part[k * HD + c] = s;
        }
        __syncthreads();
    }
}

// Any even head_dim up to 256, any head count and alignment: a wave takes one
// head of several rows; lanes stride over the pairs.
template <typename T>
__global__ __launch_bounds__(kW * 64) void qk_bwd_generic(QkBwdArgs a, RopeSlots tab) {
    constexpr int NP = T2H_MAX_HALF_HEAD / 64;
    const int lane = lane_id();
    const int D = a.head_dim, half = D / 2, H = a.heads, HD = H * D;
    const int which = (int)(blockIdx.x % a.tensors);
    const QkBwdTensor& t = a.t[which];
    const int64_t u = (blockIdx.x / a.tensors) * kW + (threadIdx.x >> 6);
    const int64_t blk = u / H;
    const int hh = (int)(u - blk * H);
    if (blk >= a.blocks) return;
    const T* x = static_cast<const T*>(t.x);
    const T* dy = static_cast<const T*>(t.dy);
    T* dx = static_cast<T*>(t.dx);
    const bool norm = t.gamma != nullptr;
    const PosSource src{a.coords, a.coord_cols, a.grid_res, a.pos_dim};
    float sg[NP][2] = {}, sb[NP][2] = {};
    for (int64_t r = blk; r < a.rows; r += a.blocks) {
        float gv[NP][2] = {}, xv[NP][2] = {}, w[NP][2] = {};
        float ss = 0.0f, dot = 0.0f;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int p = lane + 64 * i;
            if (p >= half) continue;
            const int64_t col = (int64_t)hh * D + 2 * p;
            float re = ld1(dy + r * a.dy_stride + col), im = ld1(dy + r * a.dy_stride + col + 1);
            if (a.use_rope) {
                float c = 1.0f, s = 0.0f;
                if (a.phases != nullptr) {
                    const int64_t l = r % a.phase_rows;
                    c = a.phases[(l * half + p) * 2];
                    s = a.phases[(l * half + p) * 2 + 1];
                } else if (tab.axis[p] >= 0) {
                    sincosf(mul_rn((float)src.at(r, tab.axis[p]), tab.freq[p]), &s, &c);
                }
                rotate_pair(re, im, c, -s);
            }
            gv[i][0] = re;
            gv[i][1] = im;
            if (norm) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    xv[i][e] = ld1(x + r * a.x_stride + col + e);
                    if (t.bias != nullptr) xv[i][e] = add_rn(xv[i][e], t.bias[col + e]);
                    ss = fmaf(xv[i][e], xv[i][e], ss);
                }
            }
        }
        if (norm) {
            ss = wave_sum(ss);
            const bool floor = ss < 1e-24f;
            const float rn = floor ? 1e12f : 1.0f / sqrtf(ss);
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int p = lane + 64 * i;
                if (p >= half) continue;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    xv[i][e] *= rn;
                    w[i][e] = gv[i][e] * t.gamma[(int64_t)hh * D + 2 * p + e] * a.rms_scale;
                    dot = fmaf(w[i][e], xv[i][e], dot);
                    sg[i][e] = fmaf(gv[i][e], xv[i][e], sg[i][e]);
                }
            }
            dot = wave_sum(dot);
            if (floor) dot = 0.0f;
#pragma unroll
            for (int i = 0; i < NP; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) gv[i][e] = fmaf(-xv[i][e], dot, w[i][e]) * rn;
        }
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int p = lane + 64 * i;
            if (p >= half) continue;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                sb[i][e] += gv[i][e];
                st1(dx + r * a.dx_stride + (int64_t)hh * D + 2 * p + e, gv[i][e]);
            }
        }
    }
    float* part = a.part + ((int64_t)which * a.blocks + blk) * 2 * HD + (int64_t)hh * D;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int p = lane + 64 * i;
        if (p >= half) continue;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (t.dgamma != nullptr) part[2 * p + e] = sg[i][e];
            if (t.dbias != nullptr) part[HD + 2 * p + e] = sb[i][e];
        }
    }
}

// dgamma and dbias from the partial rows: 64 columns per block, 16 strands of
// partial rows, joined in a fixed order.
__global__ __launch_bounds__(1024) void qk_bwd_sums(QkBwdArgs a) {
    __shared__ float s[16][64];
    const int HD = a.heads * a.head_dim;
    const int c = threadIdx.x & 63, strand = threadIdx.x >> 6;
    const int col = blockIdx.x * 64 + c;
    const int which = blockIdx.y >> 1, k = blockIdx.y & 1;
    float* out = k == 0 ? a.t[which].dgamma : a.t[which].dbias;
    if (out == nullptr) return;
    float v = 0.0f;
    if (col < HD) {
        const float* part = a.part + ((int64_t)which * a.blocks * 2 + k) * HD + col;
#pragma unroll 8
        for (int64_t b = strand; b < a.blocks; b += 16) v += part[b * 2 * HD];
    }
    s[strand][c] = v;
    __syncthreads();
    if (strand == 0 && col < HD) {
#pragma unroll
        for (int i = 1; i < 16; ++i) v += s[i][c];
        out[col] = k == 0 ? v * a.rms_scale : v;
    }
}

// Blocks (partial rows) per tensor: what the CUs hold at once, 3 each, 2 for f32
// rows (per_cu).
int64_t blocks_for(int64_t rows, int tensors, int per_cu) {
    const int64_t most = (int64_t)device_cu_count() * per_cu / tensors, need = (rows + kW - 1) / kW;
    return need < most ? need : most;
}

inline bool aligned_to(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }

// Rows of tensors that the 256 MB infinity cache holds in part are read through it;
// above that the loads that pass it by are faster (q and k, 12 heads of 128, f16:
// 302 MB in and out 65.4 -> 58.9 us, 453 MB 93.5 -> 92.0, 604 MB 122.5 -> 127.5; 4,096
// rows of 16 heads of 64 18.5 -> 17.1). The stores always pass it by (the other way
// 201,436 rows 683 -> 735 us).
constexpr int64_t kCachedBytes = int64_t(400) << 20;

template <typename T, int D, int NG>
void launch_fast(const QkBwdArgs& a, const RopeSlots& tab, hipStream_t s) {
    const dim3 grid((unsigned)(a.blocks * a.tensors)), block(kW * 64);
    if (3 * a.tensors * a.rows * a.heads * D * (int64_t)sizeof(T) <= kCachedBytes)
        hipLaunchKernelGGL((qk_bwd_kernel<T, D, NG, kW, false, true>), grid, block, 0, s, a, tab);
    else hipLaunchKernelGGL((qk_bwd_kernel<T, D, NG, kW, false, false>), grid, block, 0, s, a, tab);
}

template <typename T>
hipError_t launch_typed(const QkBwdArgs& a, const RopeSlots& tab, hipStream_t s) {
    // 16-byte pieces per lane, or D / 16 elements where that is less
    const int E = sizeof(T) == 2 && a.head_dim == 64 ? 8 : a.head_dim / 16;
    const int chunk = E * (int)sizeof(T) < 16 ? E * (int)sizeof(T) : 16;
    const int64_t ea = chunk > 0 ? chunk / (int)sizeof(T) : 1;
    bool fast = a.heads <= 16 && (a.head_dim == 64 || a.head_dim == 128) && a.x_stride % ea == 0 &&
                a.dy_stride % ea == 0 && a.dx_stride % ea == 0 && aligned_to(a.phases, 16);
    for (int i = 0; fast && i < a.tensors; ++i)
        fast = aligned_to(a.t[i].x, chunk) && aligned_to(a.t[i].dy, chunk) && aligned_to(a.t[i].dx, chunk) &&
               aligned_to(a.t[i].gamma, 16) && aligned_to(a.t[i].bias, 16);
    if (a.rows == 0) {
        // nothing but the sums, of no partial rows
    } else if (fast && a.rows <= kShort) {
        // both tensors of 16 heads of 64 (bf16), replayed, against two launches:
        // 1 row 6.5 -> 3.5 us, 37 rows 7.0 -> 6.4, 48 rows 6.9 -> 7.4 and 64 rows
        // 7.0 -> 8.8; eagerly every call saves another 2.5 us of launching
        const int hpi = sizeof(T) == 2 && a.head_dim == 64 ? 8 : 4;
        const dim3 grid((unsigned)((a.heads + hpi - 1) / hpi * a.tensors));
        if (a.head_dim == 128) hipLaunchKernelGGL((qk_bwd_kernel<T, 128, 1, kShortW, true, true>), grid, dim3(kShortW * 64), 0, s, a, tab);
        else hipLaunchKernelGGL((qk_bwd_kernel<T, 64, 1, kShortW, true, true>), grid, dim3(kShortW * 64), 0, s, a, tab);
        return hipGetLastError();
    } else if (!fast) {
        const int64_t units = a.blocks * a.heads;
        hipLaunchKernelGGL((qk_bwd_generic<T>), dim3((unsigned)((units + kW - 1) / kW * a.tensors)), dim3(kW * 64), 0, s, a, tab);
    } else if (a.head_dim == 128) {
        switch ((a.heads + 3) / 4) {
            case 1: launch_fast<T, 128, 1>(a, tab, s); break;
            case 2: launch_fast<T, 128, 2>(a, tab, s); break;
            case 3: launch_fast<T, 128, 3>(a, tab, s); break;
            default: launch_fast<T, 128, 4>(a, tab, s);
        }
    } else if constexpr (sizeof(T) == 2) {
        if (a.heads <= 8) launch_fast<T, 64, 1>(a, tab, s);
        else launch_fast<T, 64, 2>(a, tab, s);
    } else {
        switch ((a.heads + 3) / 4) {
            case 1: launch_fast<T, 64, 1>(a, tab, s); break;
            case 2: launch_fast<T, 64, 2>(a, tab, s); break;
            case 3: launch_fast<T, 64, 3>(a, tab, s); break;
            default: launch_fast<T, 64, 4>(a, tab, s);
        }
    }
    bool sums = false;
    for (int i = 0; i < a.tensors; ++i) sums |= a.t[i].dgamma != nullptr || a.t[i].dbias != nullptr;
    if (sums)
        hipLaunchKernelGGL(qk_bwd_sums, dim3((unsigned)((a.heads * a.head_dim + 63) / 64), (unsigned)(2 * a.tensors)), dim3(1024), 0, s, a);
    return hipGetLastError();
}

}  // namespace

int64_t qk_bwd_bytes(int64_t rows, int32_t heads, int32_t head_dim, int32_t tensors) {
    return blocks_for(rows, tensors, 3) * tensors * 2 * heads * head_dim * 4;
}

hipError_t launch_qk_bwd(QkBwdArgs a, const RopeSlots& tab, hipStream_t s) {
    a.blocks = blocks_for(a.rows, a.tensors, a.dtype == T2H_F32 ? 2 : 3);
    switch (a.dtype) {
        case T2H_F32: return launch_typed<float>(a, tab, s);
        case T2H_F16: return launch_typed<_Float16>(a, tab, s);
        default: return launch_typed<__bf16>(a, tab, s);
    }
}

}  // namespace t2h
