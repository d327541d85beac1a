// Sliding-window attention with sinks over packed qkv rows: forward and backward.
//
//   S = scale q k^T, key j visible to query i  <=>  j <= i + right  and  (j >= i - left  or  j < sinks),  0 <= j < length
//   P = softmax of S over the visible keys,  O = P V
//   dV = P^T dO,  dS = P * (dO V^T - rowsum(dO * O)),  dQ = scale dS K,  dK = scale dS^T Q
//
// Rows are [H query heads | KV key heads | KV value heads] x hd, `ld` elements apart; H is a multiple of KV and query head h reads key
// head h / (H / KV).  Sequences are L rows each or, with `offsets`, ragged.  Every query sees itself, so no softmax row is empty.
//
// One pass over the visible keys with the running maximum and sum of the softmax; the tiles that no query of the block sees are never
// read.  Operands are swapped (S^T = K Q^T): a query sits on a lane, its scores in that lane's accumulator registers, so the row
// statistics are in-lane reductions plus one exchange with lane ^ 32, and P^T feeds the next product as it lies in the registers.
// bf16 runs on v_mfma_f32_32x32x16_bf16, float32 on v_mfma_f32_32x32x2_f32 (full float32 products): an operand fragment is 16 bytes
// per lane in both, so the tile layout and the address arithmetic are shared.
#include "common.h"
#include <atomic>
#ifndef DQ_OCC
#define DQ_OCC 2
#endif
#ifndef DKV_OCC
#define DKV_OCC 1
#endif

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(4))) short short4_t;
typedef __attribute__((ext_vector_type(8))) short short8_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;
typedef __attribute__((ext_vector_type(16))) float f32x16_t;

#define WT 256                    // threads of a block: four waves of 32 queries (backward of K and V: 32 keys)
#define WROWS 128
#define LOG2E 1.4426950408889634f
#define RESCALE_TH 8.0f           // log2 units: the reference maximum is raised only when a row exceeds it by 2^8 (float32 sums: no loss)

template <typename T, int HD, int ROWS = sizeof(T) == 2 ? 64 : 32> struct WCfg {
    using Type = T;
    static constexpr int HDIM = HD;
    static constexpr int ES = sizeof(T);
    static constexpr int RB = HD * ES;                      // row bytes of a tile image
    static constexpr int CH = RB / 16;                      // 16-byte chunks per row
    static constexpr int FR = CH / 2;                       // operand fragments over the head dim (a lane half takes every other chunk)
    static constexpr int DB = HD >= 32 ? HD / 32 : 1;       // 32-row blocks of d in the transposed products
    static constexpr int KT = ROWS;                         // rows of a tile
    static constexpr int KB = KT / 32;
    static constexpr int TILE = KT * RB;
    static constexpr int NLD = (KT * CH + WT - 1) / WT;     // 16-byte loads of a thread per tile
    // rows per 256 bytes of LDS: the chunk index is XORed with the row's number inside that, so that 16 lanes reading one chunk of 16
    // successive rows (or one row's 16 chunks) touch all banks once
    static constexpr int SH = RB >= 256 ? 0 : (RB == 128 ? 1 : (RB == 64 ? 2 : 3));
    static constexpr int XM = CH < 16 ? CH - 1 : 15;
    static __device__ __forceinline__ int swizzle(int row) {
        if constexpr (CH == 2) return (row >> 2) & 1;
        else if constexpr (CH == 4) return (row & 2) | ((row >> 2) & 1);
        else return ((row & 3) << 1) | ((row >> 2) & 1);
    }
};

template <typename T, int HD> __device__ __forceinline__ int img_off(int row, int chunk) {
    using C = WCfg<T, HD>;
#ifndef OLD_SWZ
    return row * C::RB + ((chunk ^ C::swizzle(row)) << 4);
#endif
    return row * C::RB + ((chunk ^ ((row >> C::SH) & C::XM)) << 4);
}

template <class C> struct TileRegs { uint4 v[C::NLD]; };

// Byte offsets of a thread's 16-byte chunks inside a tile of rows `ld` elements apart, and the loads of the tile that starts at row0: buffer
// loads, whose range check makes the rows from nrows on zeros without a branch.
template <class C> struct TileAt {
    unsigned off[C::NLD];
    __device__ __forceinline__ TileAt(int64_t ld, int tid) {
#pragma unroll
        for (int i = 0; i < C::NLD; ++i) {
            const int id = tid + i * WT;
            off[i] = id < C::KT * C::CH ? (unsigned)(id / C::CH * ld * C::ES + (id % C::CH) * 16) : 0x7ffffff0u;
        }
    }
};
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void* p, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (unsigned)(bytes < 0 ? 0 : bytes > 0x7fffffe0 ? 0x7fffffe0 : bytes), 0x00020000);
}
template <class C, typename T>
__device__ __forceinline__ void load_tile(TileRegs<C>& t, const TileAt<C>& at, const T* __restrict__ base, int64_t ld, int row0, int nrows) {
    typedef __attribute__((ext_vector_type(4))) unsigned u4;
    const __amdgpu_buffer_rsrc_t rs = rows_rsrc(base + row0 * ld, ((nrows - 1 - row0) * ld + C::HDIM) * C::ES);
#pragma unroll
    for (int i = 0; i < C::NLD; ++i) t.v[i] = __builtin_bit_cast(uint4, (u4)__builtin_amdgcn_raw_buffer_load_b128(rs, at.off[i], 0, 0));
}
template <class C> __device__ __forceinline__ void store_tile(unsigned char* lds, const TileRegs<C>& t, int tid) {
#pragma unroll
    for (int i = 0; i < C::NLD; ++i) {
        const int id = tid + i * WT;
        if (id < C::KT * C::CH) *reinterpret_cast<uint4*>(lds + img_off<typename C::Type, C::HDIM>(id / C::CH, id % C::CH)) = t.v[i];
    }
}

// acc += A B^T over one 16-byte fragment of each operand (bf16: 8 + 8 elements of the two lane halves, float32: 4 + 4)
template <typename T> __device__ __forceinline__ f32x16_t mma_frag(uint4 a, uint4 b, f32x16_t c) {
    if constexpr (sizeof(T) == 2) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    } else {
        const f32x4_t x = __builtin_bit_cast(f32x4_t, a), y = __builtin_bit_cast(f32x4_t, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i], y[i], c, 0, 0, 0);
        return c;
    }
}

// acc += B A^T for the 32 rows blk .. blk+31 of an image: A = the image transposed (MFMA row = column 32 db + 0..31 of the image), B = the
// 32 x 32 accumulator block s as it lies (its rows are the image's rows).  bf16: the image is read by the transposing LDS read in the row
// order in which an accumulator holds its registers; float32: register e of the two halves is one product step.
template <typename T, int HD> __device__ __forceinline__ f32x16_t mma_tr(const unsigned char* lds, int blk, int db, const f32x16_t& s, f32x16_t acc, int lane) {
    if constexpr (sizeof(T) == 2) {
        const int g = lane >> 4, i = lane & 15, h2 = g >> 1;
        const int colbyte = (db * 32 + (HD >= 32 ? (g & 1) : 0) * 16 + 4 * (i & 3)) * 2;
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
            bf16x8_t p;
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = (__bf16)s[8 * s2 + j];
            const int row = blk + 16 * s2 + 4 * h2 + (i >> 2);
            const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) short4_t*)(lds + img_off<T, HD>(row, colbyte >> 4) + (colbyte & 15)));
            const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) short4_t*)(lds + img_off<T, HD>(row + 8, colbyte >> 4) + (colbyte & 15)));
            const short8_t a = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), p, acc, 0, 0, 0);
        }
    } else {
        const int d = db * 32 + (HD >= 32 ? (lane & 31) : (lane & 15)), h2 = lane >> 5;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int row = blk + (e & 3) + 8 * (e >> 2) + 4 * h2;
            const float a = *reinterpret_cast<const float*>(lds + img_off<T, HD>(row, d >> 2) + (d & 3) * 4);
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a, s[e], acc, 0, 0, 0);
        }
    }
    return acc;
}

// row index of accumulator register e on lane half h2
__device__ __forceinline__ int acc_row(int e, int h2) { return (e & 3) + 8 * (e >> 2) + 4 * h2; }

__device__ __forceinline__ f32x16_t splat16(float v) {
    f32x16_t r;
#pragma unroll
    for (int e = 0; e < 16; ++e) r[e] = v;
    return r;
}

// maximum and sum over a lane and its partner lane ^ 32, in both
__device__ __forceinline__ float pair_max(float v) {
    typedef __attribute__((ext_vector_type(2))) unsigned u2;
    const u2 x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __builtin_elementwise_maximum(__uint_as_float(x[0]), __uint_as_float(x[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
    typedef __attribute__((ext_vector_type(2))) unsigned u2;
    const u2 x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}
// orders a wave's own LDS writes and reads (its lanes exchange data without a block barrier)
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// [d][32 lanes' rows] accumulator -> a row of T per lane (both halves of a lane pair hold parts of the same row)
template <typename T, int HD> __device__ __forceinline__ void store_rows(const f32x16_t (&acc)[WCfg<T, HD>::DB], float mul, T* __restrict__ row, int h2) {
#pragma unroll
    for (int db = 0; db < WCfg<T, HD>::DB; ++db)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int d = db * 32 + 8 * t + 4 * h2;
            if (d < HD) {
                const float v[4] = {acc[db][4 * t] * mul, acc[db][4 * t + 1] * mul, acc[db][4 * t + 2] * mul, acc[db][4 * t + 3] * mul};
                st4(row + d, v);
            }
        }
}

struct WArgs {
    const void* qkv;
    const int64_t* offsets;
    void* out;
    float* lse;
    const void* dout;
    void* dqkv;
    float* delta;            // [H, R] row dots
    float* far_ws;           // [NB, KV, far_groups, far_parts] partial sums of 32 sink keys
    int64_t ld, R;
    int NB, L, H, KV, left, right, sinks;
    float scale;
    int far_groups, far_parts;
};

// rows of sequence b.  The device-side offsets cannot be checked by the host: whatever they hold, rows stay inside [0, R) and a
// sequence inside L rows.
__device__ __forceinline__ int seq_rows(const WArgs& a, int b, int64_t& start) {
    if (!a.offsets) {
        start = (int64_t)b * a.L;
        return a.L;
    }
    int64_t s = a.offsets[b], e = a.offsets[b + 1];
    s = s < 0 ? 0 : (s > a.R ? a.R : s);
    e = e < s ? s : (e > a.R ? a.R : e);
    start = s;
    return (int)(e - s > a.L ? a.L : e - s);
}

__device__ __forceinline__ bool visible(int i, int j, int left, int right, int sinks) { return j <= i + right && (j >= i - left || j < sinks); }

// the key tiles that queries [q0, q1] see: `ns` leading tiles (sinks in front of the window), then tiles w0 .. w0 + count - ns - 1
template <int KT> __device__ __forceinline__ int key_tiles(int q0, int q1, int len, int left, int right, int sinks, int& ns, int& w0) {
    const int lo = max(0, q0 - left), hi = min(len - 1, q1 + right);
    w0 = lo / KT;
    ns = min((min(sinks, len) + KT - 1) / KT, w0);
    return ns + hi / KT - w0 + 1;
}

// The K and V tiles are double-buffered in LDS: while one pair is worked on the next is on its way through registers, K first (written
// before the softmax), then V, so that only one image's worth of registers is held; one barrier per tile.
template <typename T, int HD>
__global__ __launch_bounds__(WT, (sizeof(T) * HD >= 512 ? 1 : 2)) void window_fwd_kernel(WArgs a) {
    using C = WCfg<T, HD>;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int nrb = (a.L + WROWS - 1) / WROWS;
    const int work = xcd_remap(blockIdx.x, gridDim.x);      // the row blocks of one head run on one XCD and share its L2
    const int rblk = nrb - 1 - work % nrb, h = (work / nrb) % a.H, b = work / (nrb * a.H);
    int64_t start;
    const int len = seq_rows(a, b, start);
    if (rblk * WROWS >= len) return;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, h2 = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hk = a.H + h / (a.H / a.KV);
    const T* base = (const T*)a.qkv + start * a.ld;
    const T *kb_ = base + hk * HD, *vb_ = kb_ + a.KV * HD;
    const int q0 = rblk * WROWS + wave * 32, q = q0 + r;
    const float c = a.scale * LOG2E;

    uint4 qf[C::FR];
#pragma unroll
    for (int j = 0; j < C::FR; ++j) {
        qf[j] = make_uint4(0, 0, 0, 0);
        if (q < len) qf[j] = *reinterpret_cast<const uint4*>(base + (int64_t)q * a.ld + h * HD + (2 * j + h2) * (16 / C::ES));
    }
    f32x16_t o[C::DB];
#pragma unroll
    for (int db = 0; db < C::DB; ++db) o[db] = splat16(0.f);
    float m = -INFINITY, l = 0.f;       // the lane pair holds one row's statistics: m in both, l as two partial sums

    int ns, w0;
    const int nt = key_tiles<C::KT>(rblk * WROWS, min(rblk * WROWS + WROWS, len) - 1, len, a.left, a.right, a.sinks, ns, w0);
    const int qlast = min(q0 + 31, len - 1);
    int t = ns > 0 ? 0 : w0;
    const TileAt<C> at(a.ld, tid);
    TileRegs<C> regs;
    load_tile(regs, at, kb_, a.ld, t * C::KT, len);
    store_tile(smem, regs, tid);
    load_tile(regs, at, vb_, a.ld, t * C::KT, len);
    store_tile(smem + C::TILE, regs, tid);
    __syncthreads();
    for (int it = 0; it < nt; ++it) {
        const unsigned char *kl = smem + (it & 1) * 2 * C::TILE, *vl = kl + C::TILE;
        unsigned char* next = smem + (~it & 1) * 2 * C::TILE;
        const int k0 = t * C::KT, k1 = k0 + C::KT - 1;
        const bool more = it + 1 < nt;
        t = it + 1 < ns ? it + 1 : w0 + it + 1 - ns;
        if (more) load_tile(regs, at, kb_, a.ld, t * C::KT, len);
        const bool mine = !(q0 >= len || k0 > qlast + a.right || (k1 < q0 - a.left && k0 >= a.sinks));      // this wave sees some of the tile
        f32x16_t s[C::KB];
        if (mine) {
#pragma unroll
            for (int kb = 0; kb < C::KB; ++kb) {
                s[kb] = splat16(0.f);
#pragma unroll
                for (int j = 0; j < C::FR; ++j)
                    s[kb] = mma_frag<T>(*reinterpret_cast<const uint4*>(kl + img_off<T, HD>(kb * 32 + r, 2 * j + h2)), qf[j], s[kb]);
            }
        }
        if (more) {
            store_tile(next, regs, tid);
            load_tile(regs, at, vb_, a.ld, t * C::KT, len);
        }
        if (mine) {
            if (!(k1 < len && k1 <= q0 + a.right && (k0 >= qlast - a.left || k1 < a.sinks))) {      // a border runs through the tile
#pragma unroll
                for (int kb = 0; kb < C::KB; ++kb)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int key = k0 + kb * 32 + acc_row(e, h2);
                        if (key >= len || !visible(q, key, a.left, a.right, a.sinks)) s[kb][e] = -INFINITY;
                    }
            }
            float mx = s[0][0];
#pragma unroll
            for (int kb = 0; kb < C::KB; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e) mx = __builtin_elementwise_maximum(mx, s[kb][e]);
            mx = pair_max(mx);
            if (__builtin_amdgcn_ballot_w64((mx - m) * c > RESCALE_TH) != 0) {
                const float mn = fmaxf(m, mx);
                const float alpha = mn == m ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * c);       // a row that saw nothing yet: m = mn = -inf
                m = mn;
                l *= alpha;
#pragma unroll
                for (int db = 0; db < C::DB; ++db)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[db][e] *= alpha;
            }
            const float mc = m == -INFINITY ? 0.f : m * c;
            float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kb = 0; kb < C::KB; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    s[kb][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][e], c, -mc));
                    ls[e & 3] += s[kb][e];
                }
            l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
#pragma unroll
            for (int kb = 0; kb < C::KB; ++kb)
#pragma unroll
                for (int db = 0; db < C::DB; ++db) o[db] = mma_tr<T, HD>(vl, kb * 32, db, s[kb], o[db], lane);
        }
        if (more) store_tile(next + C::TILE, regs, tid);
        __syncthreads();
    }
    if (q < len) {
        l = pair_sum(l);
        store_rows<T, HD>(o, 1.0f / l, (T*)a.out + (start + q) * a.H * HD + h * HD, h2);
        if (a.lse && h2 == 0) a.lse[(int64_t)h * a.R + start + q] = m * c + log2f(l);
    }
}

// dQ, the query on the lane; also delta = rowsum(dO * O), which the dK/dV kernels launched behind this one read
template <typename T, int HD>
__global__ __launch_bounds__(WT, (sizeof(T) * HD >= 512 ? 1 : DQ_OCC)) void window_dq_kernel(WArgs a) {
    using C = WCfg<T, HD>;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int nrb = (a.L + WROWS - 1) / WROWS;
    const int work = xcd_remap(blockIdx.x, gridDim.x);
    const int rblk = nrb - 1 - work % nrb, h = (work / nrb) % a.H, b = work / (nrb * a.H);
    int64_t start;
    const int len = seq_rows(a, b, start);
    if (rblk * WROWS >= len) return;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, h2 = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hk = a.H + h / (a.H / a.KV);
    const T* base = (const T*)a.qkv + start * a.ld;
    const T *kb_ = base + hk * HD, *vb_ = kb_ + a.KV * HD;
    const int q0 = rblk * WROWS + wave * 32, q = q0 + r;
    const float c = a.scale * LOG2E;

    uint4 qf[C::FR], gf[C::FR];
    float dl = 0.f, ls = 0.f;
#pragma unroll
    for (int j = 0; j < C::FR; ++j) {
        qf[j] = gf[j] = make_uint4(0, 0, 0, 0);
        if (q < len) {
            const int col = h * HD + (2 * j + h2) * (16 / C::ES);
            const int64_t ro = (start + q) * a.H * HD + col;
            qf[j] = *reinterpret_cast<const uint4*>(base + (int64_t)q * a.ld + col);
            gf[j] = *reinterpret_cast<const uint4*>((const T*)a.dout + ro);
            float x[4], y[4];
#pragma unroll
            for (int u = 0; u < 16 / C::ES; u += 4) {
                ld4((const T*)a.out + ro + u, x);
                ld4((const T*)a.dout + ro + u, y);
#pragma unroll
                for (int k = 0; k < 4; ++k) dl = __builtin_fmaf(x[k], y[k], dl);
            }
        }
    }
    dl = pair_sum(dl);
    if (q < len) {
        ls = a.lse[(int64_t)h * a.R + start + q];
        if (h2 == 0) a.delta[(int64_t)h * a.R + start + q] = dl;
    }
    f32x16_t dq[C::DB];
#pragma unroll
    for (int db = 0; db < C::DB; ++db) dq[db] = splat16(0.f);

    int ns, w0;
    const int nt = key_tiles<C::KT>(rblk * WROWS, min(rblk * WROWS + WROWS, len) - 1, len, a.left, a.right, a.sinks, ns, w0);
    const int qlast = min(q0 + 31, len - 1);
    int t = ns > 0 ? 0 : w0;
    const TileAt<C> at(a.ld, tid);
    TileRegs<C> regs;
    load_tile(regs, at, kb_, a.ld, t * C::KT, len);
    store_tile(smem, regs, tid);
    load_tile(regs, at, vb_, a.ld, t * C::KT, len);
    store_tile(smem + C::TILE, regs, tid);
    __syncthreads();
    for (int it = 0; it < nt; ++it) {
        const unsigned char *kl = smem + (it & 1) * 2 * C::TILE, *vl = kl + C::TILE;
        unsigned char* next = smem + (~it & 1) * 2 * C::TILE;
        const int k0 = t * C::KT, k1 = k0 + C::KT - 1;
        const bool more = it + 1 < nt;
        t = it + 1 < ns ? it + 1 : w0 + it + 1 - ns;
        const bool mine = !(q0 >= len || k0 > qlast + a.right || (k1 < q0 - a.left && k0 >= a.sinks));
        const bool whole = k1 < len && k1 <= q0 + a.right && (k0 >= qlast - a.left || k1 < a.sinks);
#pragma unroll
        for (int kb = 0; kb < C::KB; ++kb) {
            if (more) {                            // K while the first half is worked on, V while the last is
                if (kb == 0) load_tile(regs, at, kb_, a.ld, t * C::KT, len);
                if (kb == C::KB - 1) {
                    if (C::KB > 1 || !mine) store_tile(next, regs, tid);
                    if (C::KB > 1 || !mine) load_tile(regs, at, vb_, a.ld, t * C::KT, len);
                }
            }
            if (!mine) continue;
            f32x16_t s = splat16(0.f), dp = splat16(-dl);
#pragma unroll
            for (int j = 0; j < C::FR; ++j) {
                s = mma_frag<T>(*reinterpret_cast<const uint4*>(kl + img_off<T, HD>(kb * 32 + r, 2 * j + h2)), qf[j], s);
                dp = mma_frag<T>(*reinterpret_cast<const uint4*>(vl + img_off<T, HD>(kb * 32 + r, 2 * j + h2)), gf[j], dp);
            }
            if (C::KB == 1 && more) {
                store_tile(next, regs, tid);
                load_tile(regs, at, vb_, a.ld, t * C::KT, len);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], c, -ls)) * dp[e];
            if (!whole) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int key = k0 + kb * 32 + acc_row(e, h2);
                    if (key >= len || !visible(q, key, a.left, a.right, a.sinks)) s[e] = 0.f;
                }
            }
#pragma unroll
            for (int db = 0; db < C::DB; ++db) dq[db] = mma_tr<T, HD>(kl, kb * 32, db, s, dq[db], lane);
        }
        if (more) store_tile(next + C::TILE, regs, tid);
        __syncthreads();
    }
    if (q < len) store_rows<T, HD>(dq, a.scale, (T*)a.dqkv + (start + q) * (a.H + 2 * a.KV) * HD + h * HD, h2);
}

// P and dS of 32 queries (rows of the images ql and gl at qb) x 32 keys (kf, vf), and their products into dV and dK
template <class C, typename T, int HD, class VIS>
__device__ __forceinline__ void dkv_block(const unsigned char* ql, const unsigned char* gl, const float* lsl, const float* dll, int qb, const uint4 (&kf)[C::FR],
                                          const uint4 (&vf)[C::FR], float c, bool whole, VIS vis, f32x16_t (&dk)[C::DB], f32x16_t (&dv)[C::DB], int lane) {
    const int r = lane & 31, h2 = lane >> 5;
    f32x16_t s = splat16(0.f), dp = splat16(0.f);
#pragma unroll
    for (int j = 0; j < C::FR; ++j) {
        s = mma_frag<T>(*reinterpret_cast<const uint4*>(ql + img_off<T, HD>(qb + r, 2 * j + h2)), kf[j], s);
        dp = mma_frag<T>(*reinterpret_cast<const uint4*>(gl + img_off<T, HD>(qb + r, 2 * j + h2)), vf[j], dp);
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int i = qb + acc_row(e, h2);
        s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], c, -lsl[i]));
        dp[e] = s[e] * (dp[e] - dll[i]);
    }
    if (!whole) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (!vis(qb + acc_row(e, h2))) s[e] = dp[e] = 0.f;
    }
#pragma unroll
    for (int db = 0; db < C::DB; ++db) {
        dv[db] = mma_tr<T, HD>(gl, qb, db, s, dv[db], lane);
        dk[db] = mma_tr<T, HD>(ql, qb, db, dp, dk[db], lane);
    }
}

// dK and dV, the key on the lane: sweeps the queries that see the block's keys, for every query head of the group.  far_parts > 0: the
// queries that see a sink from beyond the window were done by window_far_kernel, and the sums start from its own.
template <typename T, int HD>
__global__ __launch_bounds__(WT, (sizeof(T) * HD >= 256 ? DKV_OCC : 2)) void window_dkv_kernel(WArgs a) {
    using C = WCfg<T, HD, (sizeof(T) == 2 && HD < 128) ? 64 : 32>;
    constexpr int STAGE = 2 * C::TILE + 2 * C::KT * 4;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int nrb = (a.L + WROWS - 1) / WROWS;
    const int work = xcd_remap(blockIdx.x, gridDim.x);
    const int rblk = work % nrb, hk = (work / nrb) % a.KV, b = work / (nrb * a.KV);
    int64_t start;
    const int len = seq_rows(a, b, start);
    if (rblk * WROWS >= len) return;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, h2 = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rep = a.H / a.KV;
    const T* base = (const T*)a.qkv + start * a.ld;
    const T *kb_ = base + (a.H + hk) * HD, *vb_ = kb_ + a.KV * HD;
    const int kb0 = rblk * WROWS, k0 = kb0 + wave * 32, key = k0 + r, klast = min(k0 + 31, len - 1);
    const int sinks = a.far_parts ? 0 : a.sinks;
    const float c = a.scale * LOG2E;

    uint4 kf[C::FR], vf[C::FR];
#pragma unroll
    for (int j = 0; j < C::FR; ++j) {
        kf[j] = vf[j] = make_uint4(0, 0, 0, 0);
        if (key < len) {
            kf[j] = *reinterpret_cast<const uint4*>(kb_ + (int64_t)key * a.ld + (2 * j + h2) * (16 / C::ES));
            vf[j] = *reinterpret_cast<const uint4*>(vb_ + (int64_t)key * a.ld + (2 * j + h2) * (16 / C::ES));
        }
    }
    f32x16_t dk[C::DB], dv[C::DB];
#pragma unroll
    for (int db = 0; db < C::DB; ++db) dk[db] = dv[db] = splat16(0.f);
    if (a.far_parts && k0 < min(a.sinks, len)) {
        const float* w = a.far_ws + ((int64_t)(b * a.KV + hk) * a.far_groups + k0 / 32) * a.far_parts * (2 * C::DB * 1024) + lane;
#pragma unroll
        for (int db = 0; db < C::DB; ++db)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                dk[db][e] = w[(db * 16 + e) * 64];
                dv[db][e] = w[((C::DB + db) * 16 + e) * 64];
            }
    }

    // queries that see a key of the block: from the first key minus right to the last key plus left, to the end where there are sinks
    const int qlo = max(0, kb0 - a.right), qhi = kb0 < sinks ? len - 1 : min(len - 1, min(kb0 + WROWS, len) - 1 + a.left);
    const int t0 = qlo / C::KT, nt = qhi / C::KT - t0 + 1, total = nt * rep;
    const int64_t gld = (int64_t)a.H * HD;
    const TileAt<C> qat(a.ld, tid), gat(gld, tid);
    const T* gb = (const T*)a.dout + start * gld;
    const float* cb = (tid < C::KT ? a.lse : a.delta) + start;        // the row constants: a thread of the first two groups of KT fetches one
    TileRegs<C> qr, gr;
    float cr = 0.f;
    int ft = 0, fh = hk * rep;            // the tile and head to fetch next
    auto fetch = [&]() {
        const int row0 = (t0 + ft) * C::KT;
        load_tile(qr, qat, base + fh * HD, a.ld, row0, len);
        load_tile(gr, gat, gb + fh * HD, gld, row0, len);
        const int row = row0 + tid % C::KT;
        cr = tid < 2 * C::KT && row < len ? cb[(int64_t)fh * a.R + row] : 0.f;
        if (++ft == nt) {
            ft = 0;
            ++fh;
        }
    };
    auto put = [&](unsigned char* st) {
        store_tile(st, qr, tid);
        store_tile(st + C::TILE, gr, tid);
        if (tid < 2 * C::KT) reinterpret_cast<float*>(st + 2 * C::TILE)[tid] = cr;
    };
    fetch();
    put(smem);
    __syncthreads();
    int ct = 0;
    for (int it = 0; it < total; ++it) {
        const unsigned char *ql = smem + (it & 1) * STAGE, *gl = ql + C::TILE;
        const float *lsl = reinterpret_cast<const float*>(gl + C::TILE), *dll = lsl + C::KT;
        const int q0 = (t0 + ct) * C::KT, q1 = q0 + C::KT - 1;
        ct = ct + 1 == nt ? 0 : ct + 1;
        if (it + 1 < total) fetch();
        if (!(k0 >= len || q1 < k0 - a.right || (q0 > klast + a.left && k0 >= sinks))) {
            const bool whole = q1 < len && q0 >= klast - a.right && (q1 <= k0 + a.left || klast < sinks);
#pragma unroll
            for (int qb = 0; qb < C::KB; ++qb)
                dkv_block<C, T, HD>(ql, gl, lsl, dll, qb * 32, kf, vf, c, whole,
                                    [&](int i) { return q0 + i < len && visible(q0 + i, key, a.left, a.right, sinks); }, dk, dv, lane);
        }
        if (it + 1 < total) put(smem + (~it & 1) * STAGE);
        __syncthreads();
    }
    if (key < len) {
        T* row = (T*)a.dqkv + (start + key) * (a.H + 2 * a.KV) * HD + (a.H + hk) * HD;
        store_rows<T, HD>(dk, a.scale, row, h2);
        store_rows<T, HD>(dv, 1.0f, row + a.KV * HD, h2);
    }
}

// The part of dK and dV that reaches the sinks from queries beyond the window (i > j + left): few keys, all queries of the sequence.  Left to
// the kernel above, the block with the sinks would sweep the whole sequence while the others are long done.  A wave takes one group of 32
// keys and one of `far_parts` slices of the (query head, 32-query tile) list, with its own images in LDS, and leaves its sums in far_ws.
template <typename T, int HD>
__global__ __launch_bounds__(WT) void window_far_kernel(WArgs a) {
    using C = WCfg<T, HD, 32>;
    constexpr int STAGE = 2 * C::TILE + 256, NL = C::CH / 2;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int lane = threadIdx.x & 63, r = lane & 31, h2 = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nblk = a.far_parts / 4;
    const int part = (blockIdx.x % nblk) * 4 + wave, grp = (blockIdx.x / nblk) % a.far_groups;
    const int hk = (blockIdx.x / (nblk * a.far_groups)) % a.KV, b = blockIdx.x / (nblk * a.far_groups * a.KV);
    int64_t start;
    const int len = seq_rows(a, b, start);
    const int k0 = grp * 32, key = k0 + r, kend = min(a.sinks, len);
    if (k0 >= kend) return;
    const int rep = a.H / a.KV;
    const T* base = (const T*)a.qkv + start * a.ld;
    const T *kb_ = base + (a.H + hk) * HD, *vb_ = kb_ + a.KV * HD;
    const float c = a.scale * LOG2E;
    uint4 kf[C::FR], vf[C::FR];
#pragma unroll
    for (int j = 0; j < C::FR; ++j) {
        kf[j] = vf[j] = make_uint4(0, 0, 0, 0);
        if (key < kend) {
            kf[j] = *reinterpret_cast<const uint4*>(kb_ + (int64_t)key * a.ld + (2 * j + h2) * (16 / C::ES));
            vf[j] = *reinterpret_cast<const uint4*>(vb_ + (int64_t)key * a.ld + (2 * j + h2) * (16 / C::ES));
        }
    }
    f32x16_t dk[C::DB], dv[C::DB];
#pragma unroll
    for (int db = 0; db < C::DB; ++db) dk[db] = dv[db] = splat16(0.f);
    const int t0 = (k0 + a.left + 1) / 32, nt = max(0, (len - 1) / 32 - t0 + 1);         // empty where the window reaches the end
    const int total = nt * rep, per = (total + a.far_parts - 1) / a.far_parts, i0 = part * per, i1 = min(total, i0 + per);
    unsigned char *ql = smem + wave * STAGE, *gl = ql + C::TILE;
    float *lsl = reinterpret_cast<float*>(gl + C::TILE), *dll = lsl + 32;
    const int lim = min(kend - 1, k0 + 31) + a.left;        // queries past this see every key of the group
    for (int it = i0; it < i1; ++it) {
        const int h = hk * rep + it / nt, q0 = (t0 + it % nt) * 32;
        const T *qs = base + h * HD, *gs = (const T*)a.dout + start * a.H * HD + h * HD;
        uint4 qr[NL], gr[NL];
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int id = lane + i * 64, row = q0 + id / C::CH, col = (id % C::CH) * (16 / C::ES);
            qr[i] = gr[i] = make_uint4(0, 0, 0, 0);
            if (row < len) {
                qr[i] = *reinterpret_cast<const uint4*>(qs + (int64_t)row * a.ld + col);
                gr[i] = *reinterpret_cast<const uint4*>(gs + (int64_t)row * a.H * HD + col);
            }
        }
        const float cr = q0 + r < len ? (h2 ? a.delta : a.lse)[(int64_t)h * a.R + start + q0 + r] : 0.f;
        wave_sync();                                        // the previous tile's reads are done
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int id = lane + i * 64, at = img_off<T, HD>(id / C::CH, id % C::CH);
            *reinterpret_cast<uint4*>(ql + at) = qr[i];
            *reinterpret_cast<uint4*>(gl + at) = gr[i];
        }
        lsl[lane] = cr;
        wave_sync();
        dkv_block<C, T, HD>(ql, gl, lsl, dll, 0, kf, vf, c, q0 > lim && q0 + 31 < len && kend >= k0 + 32,
                            [&](int i) { return q0 + i < len && key < kend && q0 + i > key + a.left; }, dk, dv, lane);
    }
    float* w = a.far_ws + (((int64_t)(b * a.KV + hk) * a.far_groups + grp) * a.far_parts + part) * (2 * C::DB * 1024) + lane;
#pragma unroll
    for (int db = 0; db < C::DB; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            w[(db * 16 + e) * 64] = dk[db][e];
            w[((C::DB + db) * 16 + e) * 64] = dv[db][e];
        }
}

// the parts of a group of sinks, added in their order into the first
__global__ __launch_bounds__(WT) void window_far_fold_kernel(float* __restrict__ ws, int parts, int size) {
    const int i = blockIdx.x * WT + threadIdx.x;
    float* w = ws + (int64_t)blockIdx.y * parts * size;
    if (i >= size) return;
    float t = 0.f;
#pragma unroll 8
    for (int p = 0; p < parts; ++p) t += w[(int64_t)p * size + i];
    w[i] = t;
}

// ------------------------------------------------------------------------------------------------------
template <void (*KERNEL)(WArgs)> static int launch(const char* who, int64_t blocks, size_t lds, const WArgs& a, hipStream_t s) {
    if (lds > 64 * 1024) {
        static std::atomic<unsigned long long> done{0};          // a bit per device, set once the attribute is
        int dev = 0;
        (void)hipGetDevice(&dev);
        const unsigned long long bit = 1ull << (dev & 63);
        if (!(done.load() & bit)) {
            const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (e != hipSuccess) return star_set_error(-2, "%s: %s", who, hipGetErrorString(e));
            done.fetch_or(bit);
        }
    }
    hipLaunchKernelGGL(KERNEL, dim3((unsigned)blocks), dim3(WT), lds, s, a);
    STAR_LAUNCH_CHECK(who);
    return 0;
}
template <typename T, int HD> static int run_fwd(const WArgs& a, hipStream_t s) {
    return launch<window_fwd_kernel<T, HD>>("star_attn_window_fwd", (int64_t)cdiv(a.L, WROWS) * a.H * a.NB, 4 * WCfg<T, HD>::TILE, a, s);
}
template <typename T, int HD> static int run_bwd(const WArgs& a, hipStream_t s) {
    const char* who = "star_attn_window_bwd";
    const int64_t nrb = cdiv(a.L, WROWS);
    if (int rc = launch<window_dq_kernel<T, HD>>(who, nrb * a.H * a.NB, 4 * WCfg<T, HD>::TILE, a, s)) return rc;
    if (a.far_parts) {
        const int lists = a.NB * a.KV * a.far_groups, size = 2 * WCfg<T, HD>::DB * 1024;
        if (int rc = launch<window_far_kernel<T, HD>>(who, (int64_t)lists * (a.far_parts / 4), 4 * (2 * WCfg<T, HD, 32>::TILE + 256), a, s)) return rc;
        hipLaunchKernelGGL(window_far_fold_kernel, dim3(size / WT, lists), dim3(WT), 0, s, a.far_ws, a.far_parts, size);
        STAR_LAUNCH_CHECK(who);
    }
    using C = WCfg<T, HD, (sizeof(T) == 2 && HD < 128) ? 64 : 32>;
    return launch<window_dkv_kernel<T, HD>>(who, nrb * a.KV * a.NB, 2 * (2 * C::TILE + 2 * C::KT * 4), a, s);
}

// How the far queries of the sinks are cut: about eight waves per compute unit in all, no more than 64 parts to add up, and at least two
// 32-query tiles in a part.  With over 256 sinks, or very many heads, there are enough key blocks with a long sweep to fill the chip: no parts.
static void far_plan(int NB, int L, int H, int KV, int left, int sinks, int& groups, int& parts) {
    groups = parts = 0;
    sinks = sinks < L ? sinks : L;
    if (sinks <= 0 || sinks > 256 || left >= L - 1) return;
    const int64_t lists = (int64_t)NB * KV * cdiv(sinks, 32), tiles = (int64_t)(H / KV) * cdiv(L - left - 1, 32);
    if (lists > 65535) return;
    groups = cdiv(sinks, 32);
    int64_t p = cdiv(8 * (int64_t)star_num_cus(), lists);
    if (p > tiles / 2) p = tiles / 2;
    parts = p < 4 ? 4 : p > 64 ? 64 : (int)(p / 4 * 4);
}

static int window_args(const char* who, const StarAttnWindow* g, WArgs& a) {
    STAR_CHECK(g && g->qkv && g->out, "%s: null pointer", who);
    STAR_CHECK(g->dt == STAR_BF16 || g->dt == STAR_F32, "%s: dtype %d is neither STAR_BF16 nor STAR_F32", who, g->dt);
    STAR_CHECK(g->hd == 16 || g->hd == 32 || g->hd == 64 || g->hd == 128, "%s: head dim %d not in {16,32,64,128}", who, g->hd);
    STAR_CHECK(g->NB > 0 && g->L > 0 && g->H > 0 && g->KV > 0 && g->H % g->KV == 0, "%s: bad shape NB=%d L=%d H=%d KV=%d", who, g->NB, g->L, g->H, g->KV);
    STAR_CHECK(g->H <= 65536 / g->hd, "%s: %d heads of %d are over 65536 columns", who, g->H, g->hd);
    STAR_CHECK(g->L <= (1 << 28), "%s: sequences of %d rows", who, g->L);
    STAR_CHECK(g->R >= 0 && (g->offsets || g->R == (int64_t)g->NB * g->L), "%s: %lld rows for %d sequences of %d", who, (long long)g->R, g->NB, g->L);
    STAR_CHECK(g->left >= 0 && g->right >= 0 && g->sinks >= 0, "%s: left %d, right %d and sinks %d must not be negative", who, g->left, g->right, g->sinks);
    STAR_CHECK(g->scale > 0.f && g->scale < INFINITY, "%s: scale %g must be positive", who, (double)g->scale);
    const int es = g->dt == STAR_BF16 ? 2 : 4;
    STAR_CHECK(g->ld >= (int64_t)(g->H + 2 * g->KV) * g->hd && g->ld * es % 16 == 0 && (uintptr_t)g->qkv % 16 == 0,
               "%s: qkv rows of %lld elements must hold all heads and be 16-byte aligned", who, (long long)g->ld);
    STAR_CHECK(g->ld * es < (1 << 24), "%s: qkv rows %lld elements apart", who, (long long)g->ld);       // a tile's offsets are 32 bits
    STAR_CHECK((uintptr_t)g->out % 16 == 0, "%s: out must be 16-byte aligned", who);
    STAR_CHECK((int64_t)cdiv(g->L, WROWS) * g->H * g->NB < (1ll << 31), "%s: NB, H, L too large for the grid", who);
    // a bound over L says the same as L: what is left cannot overflow in i + right and i - left
    a = WArgs{g->qkv, g->offsets, g->out, g->lse, nullptr, nullptr, nullptr, nullptr, g->ld, g->R, g->NB, g->L, g->H, g->KV,
              g->left < g->L ? g->left : g->L, g->right < g->L ? g->right : g->L, g->sinks < g->L ? g->sinks : g->L, g->scale, 0, 0};
    return 0;
}

#define BY_HD(F, T)                                                                         \
    (g->hd == 16 ? F<T, 16>(a, s) : g->hd == 32 ? F<T, 32>(a, s) : g->hd == 64 ? F<T, 64>(a, s) : F<T, 128>(a, s))

extern "C" int star_attn_window_fwd(const StarAttnWindow* g, void* stream) {
    WArgs a;
    if (int rc = window_args("star_attn_window_fwd", g, a)) return rc;
    hipStream_t s = (hipStream_t)stream;
    return g->dt == STAR_BF16 ? BY_HD(run_fwd, bf16_t) : BY_HD(run_fwd, float);
}

extern "C" int64_t star_attn_window_bwd_ws(int64_t R, int NB, int L, int H, int KV, int hd, int left, int sinks) {
    if (R < 0 || NB <= 0 || L <= 0 || H <= 0 || KV <= 0 || H % KV || hd <= 0 || left < 0 || sinks < 0) return 0;
    int groups, parts;
    far_plan(NB, L, H, KV, left, sinks, groups, parts);
    return (H * R + 63) / 64 * 64 + (int64_t)NB * KV * groups * parts * 2 * 32 * (hd < 32 ? 32 : hd);
}

extern "C" int star_attn_window_bwd(const StarAttnWindow* g, void* stream) {
    WArgs a;
    if (int rc = window_args("star_attn_window_bwd", g, a)) return rc;
    STAR_CHECK(g->lse && g->dout && g->dqkv && g->ws, "star_attn_window_bwd: null pointer");
    STAR_CHECK((uintptr_t)g->dout % 16 == 0 && (uintptr_t)g->dqkv % 16 == 0, "star_attn_window_bwd: dout and dqkv must be 16-byte aligned");
    a.dout = g->dout;
    a.dqkv = g->dqkv;
    a.delta = g->ws;
    far_plan(g->NB, g->L, g->H, g->KV, g->left, g->sinks, a.far_groups, a.far_parts);
    a.far_ws = g->ws + (g->H * g->R + 63) / 64 * 64;
    hipStream_t s = (hipStream_t)stream;
    return g->dt == STAR_BF16 ? BY_HD(run_bwd, bf16_t) : BY_HD(run_bwd, float);
}
