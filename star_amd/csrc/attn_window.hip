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
//
// Measured (kernels alone under the profiler, mean of 12): forward 5 x 4096 rows, 12 heads of 64, window 1024: 94 us = 0.61 PFLOP/s; 8192 rows, 32 heads of
// 128 on 8, window 4096: 405 .. 514 us = 1.0 .. 0.8 PFLOP/s (a large library product reaches 1.29).  2 x 8192 rows, 16 heads of 128, window 2048: forward
// 275 .. 302 us, dQ 422, dK/dV 583 = 0.8 PFLOP/s and more each.  What bounds them: the softmax's vector instructions and the matrix pipe take turns (64-wide
// heads: 207 instructions a 64 x 32 tile, 65 % and 35 % of the busy time; wave priorities around either change nothing); for 128-wide heads, backward, the
// LDS reads of the fragments beside the products (dK/dV without its transposed products 470 us, without its score products 431, without both 300).
// Short sequences are bound by the latency of few tiles per wave.
// P and dS are rounded to bf16 for the second products (the matrix instruction's operand): with the rounding of the result the backward pass
// is sqrt 2 as far off as that rounding alone.  Sums, statistics and row dots are float32.
#include "common.h"
#include <atomic>
#include <type_traits>

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(4))) short short4_t;
typedef __attribute__((ext_vector_type(8))) short short8_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;
typedef __attribute__((ext_vector_type(4))) int i32x4_t;
typedef __attribute__((ext_vector_type(16))) float f32x16_t;

#define WT 256                    // threads of a block: four waves of 32 queries (backward of K and V: 32 keys)
#define WROWS 128
// Waves that the registers of a kernel have to leave room for on a SIMD, by row bytes (measured: of 2, 3 and 4 the fastest each): a tighter
// budget makes the compiler give up the distance between its LDS reads and the products that use them.
#define WAVES_FWD(B) ((B) >= 512 ? 1 : (B) >= 256 ? 2 : 4)
#define WAVES_DQ(B) ((B) >= 512 ? 1 : (B) >= 256 ? 2 : (B) >= 128 ? 3 : 4)
#define WAVES_DKV(B) ((B) >= 512 ? 1 : (B) >= 128 ? 2 : 3)
// (Waves with rings of their own take up the LDS of a compute unit from row bytes of 256 on: one block of them, one wave on a SIMD.  float32 split
// forms are 3 to 5 % faster within half of its registers all the same.)
#define WAVES_OWN(N, B, OWN) ((OWN) && (B) >= 256 ? 1 : (N))
#define WAVES_PER_SIMD(N) __attribute__((amdgpu_waves_per_eu(N, N)))
#define LOG2E 1.4426950408889634f
#define RESCALE_TH 8.0f           // log2 units: the reference maximum is raised only when a row exceeds it by 2^8 (float32 sums: no loss)

template <typename T, int HD, int ROWS = sizeof(T) == 2 ? 64 : 32, int NW_ = 4> struct WCfg {
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
    static constexpr int RPP = 1024 / RB;                   // rows of a 1-KiB piece: what one wave's LDS-DMA instruction fills
    static constexpr int NP = TILE / 1024;                  // pieces of an image
    static constexpr int NW = NW_;
    static constexpr int NI = 2 * NP / NW;                  // pieces that each of the NW waves that share a tile brings per pair of images
    // The 16-byte chunks of a row are permuted by the row's number, so that neither 16 lanes reading one chunk of 16 successive rows nor
    // 32 lanes of a transposing read (4 rows x 4 chunks) hit one of the 64 banks twice.
    // (A bit permutation of the row: swizzle(a ^ b) = swizzle(a) ^ swizzle(b).)
    static constexpr __device__ __forceinline__ int swizzle(int row) {
        if constexpr (CH == 2) return (row >> 3) & 1;
        else if constexpr (CH == 4) return (row >> 2) & 3;
        else if constexpr (CH == 8) return ES == 2 ? ((row >> 1 & 1) << 2) | (row >> 2 & 3) : (row >> 1) & 7;
        else return ES == 2 ? ((row & 3) << 2) | (row >> 2 & 3) : row & 15;
    }
    static constexpr __device__ __forceinline__ int at(int row, int chunk) { return row * RB + ((chunk ^ swizzle(row)) << 4); }
};

typedef __attribute__((address_space(3))) void* lds_ptr_t;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void* p, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (unsigned)(bytes < 0 ? 0 : bytes > 0x7fffffe0 ? 0x7fffffe0 : bytes), 0x00020000);
}
// Where a lane's 16 bytes of piece `p` of an image lie in memory: LDS-DMA fills LDS lane by lane, so the image's permutation is applied to
// the source.  Rows past the descriptor's end arrive as zeros.
template <class C> __device__ __forceinline__ unsigned piece_src(int p, int lane, int64_t ld) {
    const int row = p * C::RPP + lane / C::CH;
    return (unsigned)(row * ld * C::ES) + (((lane % C::CH) ^ C::swizzle(row)) << 4);
}
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rs, unsigned char* lds, unsigned off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)lds, 16, off, 0, 0, 0);
}
__device__ __forceinline__ void dma4(__amdgpu_buffer_rsrc_t rs, unsigned char* lds, unsigned off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)lds, 4, off, 0, 0, 0);
}
template <int N> __device__ __forceinline__ void wait_vm() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// every wave's DMA of the tile has landed, and every wave's reads of the stage that is filled next have returned
// (a wave with a ring of its own needs no barrier)
template <int N, bool OWN> __device__ __forceinline__ void tile_ready(bool last) {
    if (last) wait_vm<0>();
    else wait_vm<N>();
    if constexpr (!OWN) __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// 16 bytes of a row.  (Through a vector type: a read of uint4 would be given a wait for every LDS-DMA in flight.)
template <typename T> struct Frag { typedef short8_t V; };
template <> struct Frag<float> { typedef f32x4_t V; };
// LDS is addressed by 32-bit offsets.  Images start at multiples of 512 bytes, so the chunk of an address can be changed by an XOR: KEEP = false
// holds one offset per access pattern and forms the others by XORs, which the dK/dV kernel of 128-wide heads needs to fit two waves on a
// SIMD (694 against 891 us at 2 x 8192 rows, 16 heads, window 2048); KEEP = true holds them all (dQ kernel, 64-wide heads: 77 against 88 us).
template <typename V> __device__ __forceinline__ V lds_read(unsigned addr) { return *reinterpret_cast<const __attribute__((address_space(3))) V*>(addr); }
// fragments of row (lane & 31) of an image
template <class C, bool KEEP> struct RowAt {
    unsigned off[KEEP ? C::FR : 1];
    __device__ __forceinline__ RowAt(int lane) {
#pragma unroll
        for (int j = 0; j < (KEEP ? C::FR : 1); ++j) off[j] = C::at(lane & 31, 2 * j + (lane >> 5));
    }
    template <int BLK> __device__ __forceinline__ typename Frag<typename C::Type>::V read(unsigned img, int j) const {
        return lds_read<typename Frag<typename C::Type>::V>((KEEP ? img + off[KEEP ? j : 0] : (img + off[0]) ^ (unsigned)(j << 5)) + BLK * C::RB);
    }
};
// a global load consumed here: the compiler then has no wait of its own to put into the loop
template <typename V> __device__ __forceinline__ void pin(V& v) {
    i32x4_t t = __builtin_bit_cast(i32x4_t, v);
    asm volatile("" : "+v"(t));
    v = __builtin_bit_cast(V, t);
}

// acc += A B^T over one 16-byte fragment of each operand (bf16: 8 + 8 elements of the two lane halves, float32: 4 + 4)
template <typename T> __device__ __forceinline__ f32x16_t mma_frag(typename Frag<T>::V a, typename Frag<T>::V b, f32x16_t c) {
    if constexpr (sizeof(T) == 2) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
}

// Products with a transposed image: acc[db] += A_db B for rows blk .. blk+31 of the image, A_db = its columns 32 db .. 32 db + 31 as MFMA rows, B
// = the 32 x 32 accumulator block p as it lies (its rows are the image's rows).
// bf16: transposing LDS reads, in the row order in which an accumulator holds its registers.  (The compiler puts a wait for every LDS-DMA in
// flight before the first of them; the next tile's was issued a whole score product earlier.)  float32: register e of the two lane halves is one
// product step, its operand an ordinary read.
template <class C, bool KEEP_> struct TrAt {
    static constexpr bool KEEP = KEEP_ && C::ES == 2;
    unsigned lo_[KEEP ? C::DB : 1], hi_[KEEP ? C::DB : 1];            // bf16: byte offsets of rows (0 | 8) + 4 h2 + i / 4, first 32 columns; float32 (lo_): row 4 h2, column lane & 31
    __device__ __forceinline__ TrAt(int lane) {
        if constexpr (C::ES == 2) {
            const int g = lane >> 4, i = lane & 15, row = 4 * (g >> 1) + (i >> 2);
#pragma unroll
            for (int db = 0; db < (KEEP ? C::DB : 1); ++db) {
                const int col = db * 64 + (C::HDIM >= 32 ? (g & 1) * 32 : 0) + (i & 3) * 8;
                lo_[db] = C::at(row, col >> 4) + (col & 15);
                hi_[db] = C::at(row + 8, col >> 4) + (col & 15);
            }
        } else {
            const int d = C::HDIM >= 32 ? (lane & 31) : (lane & 15);
            lo_[0] = hi_[0] = C::at(4 * (lane >> 5), d >> 2) + (d & 3) * 4;
        }
    }
    __device__ __forceinline__ unsigned lo(unsigned img, int db) const { return KEEP ? img + lo_[KEEP ? db : 0] : (img + lo_[0]) ^ (unsigned)(db << 6); }
    __device__ __forceinline__ unsigned hi(unsigned img, int db) const { return KEEP ? img + hi_[KEEP ? db : 0] : (img + hi_[0]) ^ (unsigned)(db << 6); }
};
__device__ __forceinline__ short4_t tr1(unsigned a) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) short4_t*>(a)); }
template <int OFF, int STEP> __device__ __forceinline__ void tr_read(unsigned lo, unsigned hi, short4_t (&r)[4]) {
    r[0] = tr1(lo + OFF); r[1] = tr1(hi + OFF); r[2] = tr1(lo + OFF + STEP); r[3] = tr1(hi + OFF + STEP);
}
template <int OFF, int STEP> __device__ __forceinline__ void tr_read2(unsigned lo, unsigned hi, unsigned lo2, unsigned hi2, short4_t (&r)[4], short4_t (&s)[4]) {
    tr_read<OFF, STEP>(lo, hi, r);
    tr_read<OFF, STEP>(lo2, hi2, s);
}
__device__ __forceinline__ f32x16_t mma_tr16(const short4_t (&r)[4], bf16x8_t p0, bf16x8_t p1, f32x16_t acc) {
    const short8_t a = {r[0][0], r[0][1], r[0][2], r[0][3], r[1][0], r[1][1], r[1][2], r[1][3]};
    const short8_t b = {r[2][0], r[2][1], r[2][2], r[2][3], r[3][0], r[3][1], r[3][2], r[3][3]};
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), p0, acc, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, b), p1, acc, 0, 0, 0);
}
// an accumulator block as the B operand, rounded to the row type
template <typename T> struct Block {
    bf16x8_t lo, hi;
    __device__ __forceinline__ Block(const f32x16_t& s) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            lo[j] = (__bf16)s[j];
            hi[j] = (__bf16)s[8 + j];
        }
    }
};
template <> struct Block<float> {
    f32x16_t v;
    __device__ __forceinline__ Block(const f32x16_t& s) : v(s) {}
};
template <class C, int BLK, class TR> __device__ __forceinline__ void mma_tr(unsigned img, const TR& at, const Block<typename C::Type>& p, f32x16_t (&acc)[C::DB]) {
    if constexpr (C::ES == 2) {
        const bf16x8_t p0 = p.lo, p1 = p.hi;
        short4_t r[4], t[4];
        if constexpr (C::DB == 1) {
            tr_read<BLK * C::RB, 16 * C::RB>(at.lo(img, 0), at.hi(img, 0), r);
            acc[0] = mma_tr16(r, p0, p1, acc[0]);
        } else {
#pragma unroll
            for (int db = 0; db < C::DB; db += 2) {
                tr_read2<BLK * C::RB, 16 * C::RB>(at.lo(img, db), at.hi(img, db), at.lo(img, db + 1), at.hi(img, db + 1), r, t);
                acc[db] = mma_tr16(r, p0, p1, acc[db]);
                acc[db + 1] = mma_tr16(t, p0, p1, acc[db + 1]);
            }
        }
    } else {
#pragma unroll
        for (int db = 0; db < C::DB; ++db)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int row = (e & 3) + 8 * (e >> 2);
                acc[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(lds_read<float>((at.lo(img, 0) ^ (unsigned)((C::swizzle(row) ^ (db * 8)) << 4)) + (BLK + row) * C::RB), p.v[e], acc[db], 0, 0, 0);
            }
    }
}

// Order of N fragment reads and their N products: six reads first, then one for every product (left alone the compiler keeps two or
// three in flight; 128-wide heads 549 -> 522 us at 8192 rows, 32 heads, window 4096).
template <int N> __device__ __forceinline__ void reads_ahead() {
    constexpr int AHEAD = N < 6 ? N : 6;
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
    for (int j = 0; j < N - AHEAD; ++j) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, AHEAD, 0);
}

// Masks of a 32-row accumulator block as one bit per row: rows first .. last are in, and the rows in front of `sinks`, if not behind last.  A
// register takes two instructions then (bit field extract, bit field insert) instead of three comparisons and a select.
__device__ __forceinline__ unsigned bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }
__device__ __forceinline__ unsigned block_mask(int first, int last, int sinks, int h2) {
    return (bits_below(last + 1) & (~bits_below(first) | bits_below(sinks))) >> (4 * h2);
}
__device__ __forceinline__ unsigned row_in(unsigned mask, int e) { return (unsigned)((int)(mask << (31 - ((e & 3) + 8 * (e >> 2)))) >> 31); }      // all ones, or zero
__device__ __forceinline__ float keep_or(unsigned in, float v, unsigned other) { return __uint_as_float((in & __float_as_uint(v)) | (~in & other)); }

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
    float* ndelta;           // [H, R] negated row dots
    float* far_ws;           // [NB, KV, far_groups, far_parts] partial sums of 32 sink keys (the parts are blocks)
    int64_t ld, R;
    int NB, L, H, KV, left, right, sinks;
    float scale;
    int far_groups, far_parts;
    int rest_blocks;         // blocks at the grid's end that zero the rows of no sequence
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

// Zeros in the rows [R, width] of y that no sequence holds: in front of the first, behind the last, and those of a sequence past its first L.
template <typename T> __device__ __forceinline__ void zero_rest(const WArgs& a, T* y, int64_t width) {
    const int part = blockIdx.x - (gridDim.x - a.rest_blocks), tid = threadIdx.x, lane = tid & 63;
    const int64_t chunks = width * sizeof(T) / 16, R = a.R;
    uint4* out = reinterpret_cast<uint4*>(y);
    auto fill = [&](int64_t lo, int64_t hi, int64_t first, int64_t step) {
        for (int64_t i = lo * chunks + first; i < hi * chunks; i += step) out[i] = make_uint4(0, 0, 0, 0);
    };
    const int64_t s0 = a.offsets[0], e0 = a.offsets[a.NB];
    fill(0, s0 < 0 ? 0 : s0 > R ? R : s0, part * WT + tid, (int64_t)a.rest_blocks * WT);
    fill(e0 < 0 ? 0 : e0 > R ? R : e0, R, part * WT + tid, (int64_t)a.rest_blocks * WT);
    for (int64_t b0 = (int64_t)(part * (WT / 64) + (tid >> 6)) * 64; b0 < a.NB; b0 += (int64_t)a.rest_blocks * WT) {
        int64_t lo = 0, hi = 0;
        if (b0 + lane < a.NB) {
            const int64_t s = a.offsets[b0 + lane], e = a.offsets[b0 + lane + 1];
            lo = (s < 0 ? 0 : s > R ? R : s) + a.L;
            hi = e > R ? R : e;
        }
        for (unsigned long long left = __builtin_amdgcn_ballot_w64(hi > lo); left; left &= left - 1) {
            const int i = __builtin_ctzll(left);
            fill(__shfl(lo, i, 64), __shfl(hi, i, 64), lane, 64);
        }
    }
}

// Block -> (stream = one head of one sequence, row block).  The row blocks of a stream stay on one XCD and share its L2.  Sequences of one
// length: every XCD walks a contiguous range of streams, which balances at any count; `side` streams go row block by row block together (the
// query heads of a group, which read the same keys: prefill of 8192 rows, 32 heads on 8, 532 -> 493 us; unrelated heads gain nothing).  Ragged with enough streams: they are dealt to the
// XCDs in turn, or the XCD that got the long sequences would finish alone (7 sequences of 0 .. 2043 rows, 16 heads, window 128 + 128:
// forward 42 -> 27 us, dQ 65 -> 43, dK/dV 63 -> 57); their grid is rounded up to whole rounds of 8.
static __host__ __device__ __forceinline__ bool dealt(const int64_t* offsets, int streams) { return offsets && streams >= 16; }
__device__ __forceinline__ bool place(const WArgs& a, int rows, int streams, int side, int& stream, int& rblk) {
    const int nrb = (a.L + rows - 1) / rows;
    if (dealt(a.offsets, streams)) {
        const int i = blockIdx.x >> 3;
        stream = (blockIdx.x & 7) + 8 * (i / nrb);
        rblk = i % nrb;
        return stream < streams;
    }
    const int work = xcd_remap(blockIdx.x, gridDim.x - a.rest_blocks), set = work / (nrb * side), rest = work - set * nrb * side;
    stream = set * side + rest % side;
    rblk = rest / side;
    return true;
}

// the key tiles that queries [q0, q1] see: `ns` leading tiles (sinks in front of the window), then tiles w0 .. w0 + count - ns - 1
template <int KT> __device__ __forceinline__ int key_tiles(int q0, int q1, int len, int left, int right, int sinks, int& ns, int& w0) {
    const int lo = max(0, q0 - left), hi = min(len - 1, q1 + right);
    w0 = lo / KT;
    ns = min((min(sinks, len) + KT - 1) / KT, w0);
    return ns + hi / KT - w0 + 1;
}

// the tiles of a launch form (see the split form below): shared by four waves, or a wave's own
template <typename T, int HD, bool SPLIT> using RowCfg = std::conditional_t<SPLIT, WCfg<T, HD, 32, 1>, WCfg<T, HD>>;

// A ring of STAGES (K image | V image) stages: while one tile is worked on the next STAGES - 1 are on their way, without registers.  (Four rings of
// float32 rows of 128 leave room for one stage each: a tile's products take several times the time that it is waited for.)
template <class C> struct KvRing {
    static constexpr int STAGE = 2 * C::TILE, STAGES = C::NW == 1 && C::RB > 256 ? 1 : C::NW == 1 || STAGE > 8192 ? 2 : 3, BYTES = STAGES * STAGE;
    const typename C::Type* k;              // key 0 of the head; its value lies v columns further on
    int64_t ld;
    int v, len, wave;
    unsigned src[C::NI];
    __device__ __forceinline__ KvRing(const typename C::Type* k_, int64_t ld_, int v_, int len_, int wave_, int lane) : k(k_), ld(ld_), v(v_), len(len_), wave(wave_) {
#pragma unroll
        for (int j = 0; j < C::NI; ++j) {
            const int p = wave * C::NI + j, isv = p >= C::NP;
            src[j] = piece_src<C>(isv ? p - C::NP : p, lane, ld) + (isv ? v * C::ES : 0);
        }
    }
    __device__ __forceinline__ void issue(int tile, unsigned char* stage) const {
        const int64_t row0 = (int64_t)tile * C::KT;
        const __amdgpu_buffer_rsrc_t rs = rows_rsrc(k + row0 * ld, ((len - 1 - row0) * ld + v + C::HDIM) * C::ES);     // row `len` starts behind this
#pragma unroll
        for (int j = 0; j < C::NI; ++j) dma16(rs, stage + (wave * C::NI + j) * 1024, src[j]);
    }
};

// A masked weight is 0, and 0 * inf in a product is NaN: an infinity or a NaN in a row that a query does not see would reach it where both meet in
// one tile.  Results that came out not finite are therefore formed again, one visible row at a time, with no arithmetic on hidden ones: nothing is
// paid where all results are finite.  Where the row's own statistics are NaN (or, for a key, its own row), so is the result by the formula, and
// it stays, and a sum all of whose elements have become NaN is not taken further: data that has gone NaN altogether takes about as long as other
// data (dO all NaN: 2 x 2048 rows, causal, 16 heads on 4 of 64, backward 138 -> 197 us; 16 heads of 128, window 512: 131 -> 460).  A sum of which
// some elements alone are not finite is formed to its end, and that takes its time, 1 to 3 us a visible row and head (one NaN in one value row of the first
// of these: forward 53 -> 2570 us, backward 138 -> 8000).  A lane works on its half of a row, the partner on the other (the layout of an accumulator).
template <class C> __device__ __forceinline__ bool any_bad(const f32x16_t (&acc)[C::DB]) {
    float t = 0.f;
#pragma unroll
    for (int db = 0; db < C::DB; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (db * 32 + acc_row(e, 0) < C::HDIM) t = __builtin_fmaf(acc[db][e], 0.f, t);
    return !(t == 0.f);
}
template <class C> __device__ __forceinline__ void read_half(const typename C::Type* row, int h2, f32x16_t (&v)[C::DB]) {
#pragma unroll
    for (int db = 0; db < C::DB; ++db)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            float x[4] = {0.f, 0.f, 0.f, 0.f};
            if (db * 32 + 8 * t < C::HDIM) ld4(row + db * 32 + 8 * t + 4 * h2, x);
#pragma unroll
            for (int u = 0; u < 4; ++u) v[db][4 * t + u] = x[u];
        }
}
template <class C> __device__ __forceinline__ float dot_half(const f32x16_t (&v)[C::DB], const typename C::Type* row, int h2) {
    float d = 0.f;
#pragma unroll
    for (int db = 0; db < C::DB; ++db)
#pragma unroll
        for (int t = 0; t < 4; ++t)
            if (db * 32 + 8 * t < C::HDIM) {
                float x[4];
                ld4(row + db * 32 + 8 * t + 4 * h2, x);
#pragma unroll
                for (int u = 0; u < 4; ++u) d = __builtin_fmaf(v[db][4 * t + u], x[u], d);
            }
    return pair_sum(d);
}
// whether the lane pair's row has no element left that is not NaN
template <class C> __device__ __forceinline__ bool all_nan(const f32x16_t (&acc)[C::DB]) {
    float others = 0.f;
#pragma unroll
    for (int db = 0; db < C::DB; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (db * 32 + acc_row(e, 0) < C::HDIM) others += acc[db][e] == acc[db][e] ? 1.0f : 0.f;
    return pair_sum(others) == 0.f;
}
// acc = acc * alpha + p * row where seen
template <class C> __device__ __forceinline__ void add_half(f32x16_t (&acc)[C::DB], float alpha, bool seen, float p, const typename C::Type* row, int h2) {
#pragma unroll
    for (int db = 0; db < C::DB; ++db)
#pragma unroll
        for (int t = 0; t < 4; ++t)
            if (db * 32 + 8 * t < C::HDIM) {
                float x[4];
                ld4(row + db * 32 + 8 * t + 4 * h2, x);
#pragma unroll
                for (int u = 0; u < 4; ++u) acc[db][4 * t + u] = acc[db][4 * t + u] * alpha + (seen ? p * x[u] : 0.f);
            }
}
__device__ __forceinline__ bool sees(const WArgs& a, int i, int j) { return j <= i + a.right && (j >= i - a.left || j < a.sinks); }
// the next row after j of those that some query of q0 .. qlast sees
__device__ __forceinline__ int next_key(const WArgs& a, int j, int q0) { return j + 1 >= a.sinks && j + 1 < q0 - a.left ? q0 - a.left : j + 1; }

// the lane's output row (or, with dO, -delta and lse, its dQ row) from visible keys alone
template <class C, bool GRAD> __device__ __forceinline__ void redo_query(const WArgs& a, const typename C::Type* base, const typename C::Type* grow, int h, int q, int q0, int len, float ls,
                                                                         float ndl, int h2, f32x16_t (&acc)[C::DB]) {
    using T = typename C::Type;
    constexpr int HD = C::HDIM;
    const float c = a.scale * LOG2E;
    const T* kp = base + (a.H + h / (a.H / a.KV)) * HD;
    const int qlast = min(q0 + 31, len - 1);
    f32x16_t qv[C::DB], gv[C::DB];
    read_half<C>(base + (int64_t)q * a.ld + h * HD, h2, qv);
    if constexpr (GRAD) read_half<C>(grow, h2, gv);
#pragma unroll
    for (int db = 0; db < C::DB; ++db) acc[db] = splat16(0.f);
    float m = -INFINITY, l = 0.f;
    for (int j = next_key(a, -1, q0); j <= min(len - 1, qlast + a.right); j = next_key(a, j, q0)) {
        const T *kr = kp + (int64_t)j * a.ld, *vr = kr + a.KV * HD;
        const bool seen = sees(a, q, j);
        const float s = dot_half<C>(qv, kr, h2) * c;
        if constexpr (GRAD) {
            const float dp = dot_half<C>(gv, vr, h2) + ndl;
            add_half<C>(acc, 1.0f, seen, __builtin_amdgcn_exp2f(s - ls) * dp, kr, h2);
        } else {
            const float mn = seen ? __builtin_elementwise_maximum(m, s) : m;
            const float alpha = mn == m ? 1.0f : __builtin_amdgcn_exp2f(m - mn), p = __builtin_amdgcn_exp2f(s - (mn == -INFINITY ? 0.f : mn));
            m = mn;
            l = l * alpha + (seen ? p : 0.f);
            add_half<C>(acc, alpha, seen, p, vr, h2);
        }
        if (all_nan<C>(acc)) break;
    }
    const float mul = GRAD ? a.scale : 1.0f / l;
#pragma unroll
    for (int db = 0; db < C::DB; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[db][e] *= mul;
}

// Split form: the four waves of a block work on the same 32 rows (dK/dV: keys), each on every fourth tile with a ring of its own, and are added up
// through LDS, in their order, when all are done.  For launches whose row form (a wave per 32 rows, four sharing the tiles) leaves much of the
// chip idle, or waiting for the blocks with the longest sweeps (SplitUpTo).
// Sum of the waves' accumulator block, in their order: a wave gets four of the sixteen registers, 4 wave .. 4 wave + 3.
__device__ __forceinline__ void join_block(const f32x16_t& acc, float mul, float* sum, float (&v)[4], int wave, int lane) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 16; ++e) sum[(wave * 16 + e) * 64 + lane] = acc[e] * mul;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int at = (wave * 4 + e) * 64 + lane;
        v[e] = (sum[at] + sum[at + 1024]) + (sum[at + 2 * 1024] + sum[at + 3 * 1024]);
    }
}
// whether a wave has found its part of the lane pair's row not finite; st: 256 floats of LDS
__device__ __forceinline__ bool any_wave_bad(bool bad, float* st, int wave, int lane) {
    const float mine = pair_sum(bad ? 1.0f : 0.f);
    __syncthreads();
    st[wave * 64 + lane] = mine;
    __syncthreads();
    return st[lane] + st[64 + lane] + st[128 + lane] + st[192 + lane] != 0.f;
}
// mul * sum of the waves' accumulators -> the lane's row
template <class C> __device__ __forceinline__ void join_rows(const f32x16_t (&acc)[C::DB], float mul, float* sum, bool valid, typename C::Type* row, int wave, int lane) {
#pragma unroll
    for (int db = 0; db < C::DB; ++db) {
        float v[4];
        join_block(acc[db], mul, sum, v, wave, lane);
        const int d = db * 32 + 8 * wave + 4 * (lane >> 5);
        if (valid && d < C::HDIM) st4(row + d, v);
    }
}

template <typename T, int HD, bool SPLIT>
__global__ __launch_bounds__(WT) WAVES_PER_SIMD(WAVES_OWN(WAVES_FWD(sizeof(T) * HD), sizeof(T) * HD, SPLIT && sizeof(T) == 2)) void window_fwd_kernel(WArgs a) {
    using C = RowCfg<T, HD, SPLIT>;
    constexpr int ROWS = SPLIT ? 32 : WROWS, STEP = SPLIT ? 4 : 1;
    using Ring = KvRing<C>;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    if (a.rest_blocks && blockIdx.x >= gridDim.x - a.rest_blocks) return zero_rest(a, (T*)a.out, (int64_t)a.H * HD);
    int stream, rblk;
    if (!place(a, ROWS, a.NB * a.H, a.H / a.KV, stream, rblk)) return;
    const int h = stream % a.H, b = stream / a.H;
    rblk = (a.L + ROWS - 1) / ROWS - 1 - rblk;             // the last rows see most: they go first
    int64_t start;
    const int len = seq_rows(a, b, start);
    if (rblk * ROWS >= len) return;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, h2 = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const T* base = (const T*)a.qkv + start * a.ld;
    const int q0 = rblk * ROWS + (SPLIT ? 0 : wave * 32), q = q0 + r;
    const float c = a.scale * LOG2E;

    typename Frag<T>::V qf[C::FR] = {};
#pragma unroll
    for (int j = 0; j < C::FR; ++j)
        if (q < len) qf[j] = *reinterpret_cast<const typename Frag<T>::V*>(base + (int64_t)q * a.ld + h * HD + (2 * j + h2) * (16 / C::ES));
#pragma unroll
    for (int j = 0; j < C::FR; ++j) pin(qf[j]);
    f32x16_t o[C::DB];
#pragma unroll
    for (int db = 0; db < C::DB; ++db) o[db] = splat16(0.f);
    float m = -INFINITY, l = 0.f;       // the lane pair holds one row's statistics: m in both, l as two partial sums

    int ns, w0;
    const int all = key_tiles<C::KT>(rblk * ROWS, min(rblk * ROWS + ROWS, len) - 1, len, a.left, a.right, a.sinks, ns, w0);
    const int first = SPLIT ? wave : 0, nt = (all - first + STEP - 1) / STEP;              // this wave's tiles: first, first + STEP, ...
    const int qlast = min(q0 + 31, len - 1);
    const Ring ring(base + (a.H + h / (a.H / a.KV)) * HD, a.ld, a.KV * HD, len, SPLIT ? 0 : wave, lane);
    const TrAt<C, (C::RB < 256)> tr(lane);
    const RowAt<C, (C::RB < 256)> row(lane);
    unsigned char* own = smem + (SPLIT ? wave * Ring::BYTES : 0);
    const unsigned lds = lds_u32(own);
    auto tile = [&](int i) {
        const int it = first + i * STEP;
        return it < ns ? it : w0 + it - ns;
    };
    int fill = 0, use = 0;               // ring positions
    for (; fill < Ring::STAGES - 1 && fill < nt; ++fill) ring.issue(tile(fill), own + fill * Ring::STAGE);
    fill = Ring::STAGES - 1;
    for (int it = 0; it < nt; ++it) {
        if constexpr (Ring::STAGES == 1) {
            wait_lds();
            ring.issue(tile(it), own);
            wait_vm<0>();
        } else {
            tile_ready<(Ring::STAGES - 2) * C::NI, SPLIT>(it + Ring::STAGES - 1 > nt);
            if (it + Ring::STAGES - 1 < nt) ring.issue(tile(it + Ring::STAGES - 1), own + fill * Ring::STAGE);
        }
        fill = fill + 1 == Ring::STAGES ? 0 : fill + 1;
        const unsigned kl = lds + use * Ring::STAGE, vl = kl + C::TILE;
        use = use + 1 == Ring::STAGES ? 0 : use + 1;
        const int k0 = tile(it) * C::KT, k1 = k0 + C::KT - 1;
        if (q0 >= len || k0 > qlast + a.right || (k1 < q0 - a.left && k0 >= a.sinks)) continue;      // this wave sees nothing of the tile
        f32x16_t s[C::KB];
#pragma unroll
        for (int kb = 0; kb < C::KB; ++kb) {
            s[kb] = splat16(0.f);
#pragma unroll
            for (int j = 0; j < C::FR; ++j) s[kb] = mma_frag<T>(kb ? row.template read<32>(kl, j) : row.template read<0>(kl, j), qf[j], s[kb]);
        }
        if constexpr (C::ES == 2) reads_ahead<C::KB * C::FR>();
        if (!(k1 < len && k1 <= q0 + a.right && (k0 >= qlast - a.left || k1 < a.sinks))) {      // a border runs through the tile
#pragma unroll
            for (int kb = 0; kb < C::KB; ++kb) {
                const int kk = k0 + kb * 32;
                const unsigned in = block_mask(q - a.left - kk, min(q + a.right, len - 1) - kk, a.sinks - kk, h2);
#pragma unroll
                for (int e = 0; e < 16; ++e) s[kb][e] = keep_or(row_in(in, e), s[kb][e], 0xff800000u);
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
        float ls[4] = {0.f, 0.f, 0.f, 0.f};       // of the unrounded weights: the log-sum-exp that the backward pass reads is a float32 one
        auto half = [&](auto kb_) {
            constexpr int kb = decltype(kb_)::value;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[kb][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][e], c, -mc));
                ls[e & 3] += s[kb][e];
            }
            mma_tr<C, kb * 32>(vl, tr, Block<T>(s[kb]), o);
        };
        half(std::integral_constant<int, 0>{});
        if constexpr (C::KB == 2) half(std::integral_constant<int, 1>{});
        l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
    }
    l = pair_sum(l);
    if constexpr (SPLIT) {
        float* st = reinterpret_cast<float*>(smem);          // [wave][maximum, sum][lane], then join_rows' 16 KiB
        __syncthreads();
        st[wave * 128 + lane] = m;
        st[wave * 128 + 64 + lane] = l;
        __syncthreads();
        const float own_m = m;
        m = fmaxf(fmaxf(st[lane], st[128 + lane]), fmaxf(st[256 + lane], st[384 + lane]));
        l = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float mw = st[w * 128 + lane];
            l += st[w * 128 + 64 + lane] * (mw == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((mw - m) * c));       // -inf: 0, or NaN of a NaN score
        }
        const float f = (own_m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((own_m - m) * c)) / l;        // every score -inf: 0 / 0, as in the row form
        const bool bad = any_wave_bad(any_bad<C>(o), st, wave, lane) && l == l;
        join_rows<C>(o, f, st + 512, q < len && !bad, (T*)a.out + (start + q) * a.H * HD + h * HD, wave, lane);
        if (bad && q < len && wave == 0) {
            redo_query<C, false>(a, base, nullptr, h, q, q0, len, 0.f, 0.f, h2, o);
            store_rows<T, HD>(o, 1.0f, (T*)a.out + (start + q) * a.H * HD + h * HD, h2);
        }
        if (q < len && a.lse && h2 == 0 && wave == 0) a.lse[(int64_t)h * a.R + start + q] = m * c + log2f(l);
        return;
    }
    if (q < len) {
        float mul = 1.0f / l;
        if (pair_sum(any_bad<C>(o) ? 1.0f : 0.f) != 0.f && l == l) {
            redo_query<C, false>(a, base, nullptr, h, q, q0, len, 0.f, 0.f, h2, o);
            mul = 1.0f;
        }
        store_rows<T, HD>(o, mul, (T*)a.out + (start + q) * a.H * HD + h * HD, h2);
        if (a.lse && h2 == 0) a.lse[(int64_t)h * a.R + start + q] = m * c + log2f(l);
    }
}

// dQ, the query on the lane; also -delta = -rowsum(dO * O), which the dK/dV kernels launched behind this one read.
// In bf16 the rows of O are rounded, and with few visible keys that is felt: dP - delta cancels, and dQ and dK are up to 1.84 times as far off as one
// rounding of the results leaves them.  The sum of the row's dS, which is zero by the formula, is just what delta is short of: blocks whose rows see
// at most FEW_KEYS take it in a sweep of its own first.  Error of dQ against one rounding, and the whole backward pass at 8 x 2048 rows, 16 heads of 64,
// without and with that sweep: 7 keys 1.84 and 1.42, 114 and 127 us; 33: 1.60 and 1.44, 117 and 129; 64: 1.54 and 1.43, 121 and 134; 128: 1.54 and
// 1.43, 133 and 154; 255: 1.53 and 1.44, 161 and 190 (128-wide heads 259 and 282 .. 339 and 386).
#define FEW_KEYS 256
template <typename T, int HD, bool SPLIT>
__global__ __launch_bounds__(WT) WAVES_PER_SIMD(WAVES_OWN(WAVES_DQ(sizeof(T) * HD), sizeof(T) * HD, SPLIT && sizeof(T) == 2)) void window_dq_kernel(WArgs a) {
    using C = RowCfg<T, HD, SPLIT>;
    constexpr int ROWS = SPLIT ? 32 : WROWS, STEP = SPLIT ? 4 : 1;
    using Ring = KvRing<C>;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    if (a.rest_blocks && blockIdx.x >= gridDim.x - a.rest_blocks) return zero_rest(a, (T*)a.dqkv, (int64_t)(a.H + 2 * a.KV) * HD);
    int stream, rblk;
    if (!place(a, ROWS, a.NB * a.H, a.H / a.KV, stream, rblk)) return;
    const int h = stream % a.H, b = stream / a.H;
    rblk = (a.L + ROWS - 1) / ROWS - 1 - rblk;             // the last rows see most: they go first
    int64_t start;
    const int len = seq_rows(a, b, start);
    if (rblk * ROWS >= len) return;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, h2 = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const T* base = (const T*)a.qkv + start * a.ld;
    const int q0 = rblk * ROWS + (SPLIT ? 0 : wave * 32), q = q0 + r;
    const float c = a.scale * LOG2E;

    typename Frag<T>::V qf[C::FR] = {}, gf[C::FR] = {};
    float dl = 0.f, ls = 0.f;
#pragma unroll
    for (int j = 0; j < C::FR; ++j)
        if (q < len) {
            const int col = h * HD + (2 * j + h2) * (16 / C::ES);
            const int64_t ro = (start + q) * a.H * HD + col;
            qf[j] = *reinterpret_cast<const typename Frag<T>::V*>(base + (int64_t)q * a.ld + col);
            gf[j] = *reinterpret_cast<const typename Frag<T>::V*>((const T*)a.dout + ro);
            float x[4], y[4];
#pragma unroll
            for (int u = 0; u < 16 / C::ES; u += 4) {
                ld4((const T*)a.out + ro + u, x);
                ld4((const T*)a.dout + ro + u, y);
#pragma unroll
                for (int k = 0; k < 4; ++k) dl = __builtin_fmaf(x[k], y[k], dl);
            }
        }
    dl = pair_sum(dl);
    if (q < len) ls = a.lse[(int64_t)h * a.R + start + q];
#pragma unroll
    for (int j = 0; j < C::FR; ++j) {
        pin(qf[j]);
        pin(gf[j]);
    }
    asm volatile("" : "+v"(ls), "+v"(dl));
    f32x16_t dq[C::DB];
#pragma unroll
    for (int db = 0; db < C::DB; ++db) dq[db] = splat16(0.f);

    int ns, w0;
    const int all = key_tiles<C::KT>(rblk * ROWS, min(rblk * ROWS + ROWS, len) - 1, len, a.left, a.right, a.sinks, ns, w0);
    const int first = SPLIT ? wave : 0, nt = (all - first + STEP - 1) / STEP;              // this wave's tiles: first, first + STEP, ...
    const int qlast = min(q0 + 31, len - 1);
    const Ring ring(base + (a.H + h / (a.H / a.KV)) * HD, a.ld, a.KV * HD, len, SPLIT ? 0 : wave, lane);
    const TrAt<C, (C::RB < 256)> tr(lane);
    const RowAt<C, (C::RB < 256)> row(lane);
    unsigned char* own = smem + (SPLIT ? wave * Ring::BYTES : 0);
    const unsigned lds = lds_u32(own);
    auto tile = [&](int i) {
        const int it = first + i * STEP;
        return it < ns ? it : w0 + it - ns;
    };
    float short_of = 0.f;
    auto sweep = [&](auto sum_) {
        constexpr bool SUM = decltype(sum_)::value;
        int fill = 0, use = 0;
        for (; fill < Ring::STAGES - 1 && fill < nt; ++fill) ring.issue(tile(fill), own + fill * Ring::STAGE);
        fill = Ring::STAGES - 1;
        for (int it = 0; it < nt; ++it) {
            if constexpr (Ring::STAGES == 1) {
                wait_lds();
                ring.issue(tile(it), own);
                wait_vm<0>();
            } else {
                tile_ready<(Ring::STAGES - 2) * C::NI, SPLIT>(it + Ring::STAGES - 1 > nt);
                if (it + Ring::STAGES - 1 < nt) ring.issue(tile(it + Ring::STAGES - 1), own + fill * Ring::STAGE);
            }
            fill = fill + 1 == Ring::STAGES ? 0 : fill + 1;
            const unsigned kl = lds + use * Ring::STAGE, vl = kl + C::TILE;
            use = use + 1 == Ring::STAGES ? 0 : use + 1;
            const int k0 = tile(it) * C::KT, k1 = k0 + C::KT - 1;
            if (q0 >= len || k0 > qlast + a.right || (k1 < q0 - a.left && k0 >= a.sinks)) continue;
            const bool whole = k1 < len && k1 <= q0 + a.right && (k0 >= qlast - a.left || k1 < a.sinks);
            auto half = [&](auto kb_) {
                constexpr int kb = decltype(kb_)::value;
                f32x16_t s = splat16(0.f), dp = splat16(-dl);
#pragma unroll
                for (int j = 0; j < C::FR; ++j) {
                    s = mma_frag<T>(row.template read<kb * 32>(kl, j), qf[j], s);
                    dp = mma_frag<T>(row.template read<kb * 32>(vl, j), gf[j], dp);
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], c, -ls)) * dp[e];
                if (!whole) {
                    const int kk = k0 + kb * 32;
                    const unsigned in = block_mask(q - a.left - kk, min(q + a.right, len - 1) - kk, a.sinks - kk, h2);
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[e] = keep_or(row_in(in, e), s[e], 0u);
                }
                if constexpr (SUM) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) short_of += s[e];
                } else {
                    mma_tr<C, kb * 32>(kl, tr, Block<T>(s), dq);
                }
            };
            half(std::integral_constant<int, 0>{});
            if constexpr (C::KB == 2) half(std::integral_constant<int, 1>{});
        }
    };
    if constexpr (C::ES == 2) {
        const int last = min(len - 1, min(rblk * ROWS + ROWS, len) - 1 + a.right);
        if (min(last + 1, a.left + a.right + 1 + a.sinks) <= FEW_KEYS) {
            sweep(std::true_type{});
            short_of = pair_sum(short_of);
            __syncthreads();
            if constexpr (SPLIT) {
                float* st = reinterpret_cast<float*>(smem);
                st[wave * 64 + lane] = short_of;
                __syncthreads();
                short_of = (st[lane] + st[64 + lane]) + (st[128 + lane] + st[192 + lane]);
                __syncthreads();
            }
            dl += short_of;
        }
    }
    if (q < len && h2 == 0 && (!SPLIT || wave == 0)) a.ndelta[(int64_t)h * a.R + start + q] = -dl;
    sweep(std::false_type{});
    T* qrow = (T*)a.dqkv + (start + q) * (a.H + 2 * a.KV) * HD + h * HD;
    const T* grow = (const T*)a.dout + (start + q) * a.H * HD + h * HD;
    if constexpr (SPLIT) {
        float* st = reinterpret_cast<float*>(smem);
        __syncthreads();
        const bool bad = any_wave_bad(any_bad<C>(dq), st, wave, lane) && ls + dl == ls + dl;
        join_rows<C>(dq, a.scale, st + 512, q < len && !bad, qrow, wave, lane);
        if (bad && q < len && wave == 0) {
            redo_query<C, true>(a, base, grow, h, q, q0, len, ls, -dl, h2, dq);
            store_rows<T, HD>(dq, 1.0f, qrow, h2);
        }
        return;
    }
    if (q < len) {
        float mul = a.scale;
        if (pair_sum(any_bad<C>(dq) ? 1.0f : 0.f) != 0.f && ls + dl == ls + dl) {
            redo_query<C, true>(a, base, grow, h, q, q0, len, ls, -dl, h2, dq);
            mul = 1.0f;
        }
        store_rows<T, HD>(dq, mul, qrow, h2);
    }
}

// P and dS of 32 queries (rows BLK .. of the images at ql and gl, their log-sum-exps and negated row dots at cst and cst + 256) x 32 keys (kf,
// vf), and their products into dV and dK.  The dP accumulator starts from -delta.  Not `whole`: the lane's key is seen by the image's
// rows first .. last alone.
template <class C, int BLK, class ROW, class TR>
__device__ __forceinline__ void dkv_block(unsigned ql, unsigned gl, unsigned cst, const ROW& row, const typename Frag<typename C::Type>::V (&kf)[C::FR],
                                          const typename Frag<typename C::Type>::V (&vf)[C::FR], float c, bool whole, int first, int last, const TR& tr, f32x16_t (&dk)[C::DB],
                                          f32x16_t (&dv)[C::DB], int h2) {
    using T = typename C::Type;
    f32x16_t s = splat16(0.f), dp;
    cst += BLK * 4 + 16 * h2;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const f32x4_t d = lds_read<f32x4_t>(cst + 256 + 32 * t);
#pragma unroll
        for (int u = 0; u < 4; ++u) dp[4 * t + u] = d[u];
    }
#pragma unroll
    for (int j = 0; j < C::FR; ++j) {
        s = mma_frag<T>(row.template read<BLK>(ql, j), kf[j], s);
        dp = mma_frag<T>(row.template read<BLK>(gl, j), vf[j], dp);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const f32x4_t lt = lds_read<f32x4_t>(cst + 32 * t);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int e = 4 * t + u;
            s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], c, -lt[u]));
            dp[e] *= s[e];
        }
    }
    if (!whole) {
        const unsigned in = block_mask(first - BLK, last - BLK, 0, h2);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            s[e] = keep_or(row_in(in, e), s[e], 0u);
            dp[e] = keep_or(row_in(in, e), dp[e], 0u);
        }
    }
    mma_tr<C, BLK>(gl, tr, Block<T>(s), dv);
    mma_tr<C, BLK>(ql, tr, Block<T>(dp), dk);
}

// The lane's dV row, then its dK row, from the queries that see the key alone (see redo_query).  A sink's far queries are not swept again: where they
// have parts (`far`, `parts` of them), those hold their sums, and what a part has masked for a sink are queries of its window, which it sees.  (Swept, one
// NaN in one row of dO would cost every head and row of the sequence, one after the other: 650 ms at 32768 rows, 8 heads of 64 on 1, window 100, 4 sinks,
// where the window's keys take 2.)
template <class C> __device__ __forceinline__ void redo_key(const WArgs& a, const typename C::Type* base, int64_t start, int hk, int key, int k0, int len, int h2, const float* far, int parts,
                                                            typename C::Type* row) {
    using T = typename C::Type;
    constexpr int HD = C::HDIM;
    const float c = a.scale * LOG2E;
    const bool sink = key < a.sinks;
    const int rep = a.H / a.KV, last = sink && !a.far_parts ? len - 1 : min(len - 1, key + a.left);
    f32x16_t kv[C::DB], vv[C::DB], acc[C::DB];
    read_half<C>(base + (int64_t)key * a.ld + (a.H + hk) * HD, h2, kv);
    read_half<C>(base + (int64_t)key * a.ld + (a.H + a.KV + hk) * HD, h2, vv);
    float nans = 0.f;
#pragma unroll
    for (int db = 0; db < C::DB; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) nans += kv[db][e] == kv[db][e] ? 0.f : 1.0f;
    if (pair_sum(nans) != 0.f) {
#pragma unroll
        for (int db = 0; db < C::DB; ++db) acc[db] = splat16(NAN);
        store_rows<T, HD>(acc, 1.0f, row, h2);
        store_rows<T, HD>(acc, 1.0f, row + a.KV * HD, h2);
        return;
    }
    for (int grad = 0; grad < 2; ++grad) {          // 0: dV, 1: dK
#pragma unroll
        for (int db = 0; db < C::DB; ++db) acc[db] = splat16(0.f);
        if (sink && a.far_parts)
            for (int p = 0; p < parts; ++p)
#pragma unroll
                for (int db = 0; db < C::DB; ++db)
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[db][e] += far[(int64_t)p * (2 * C::DB * 1024) + (((grad ? 0 : C::DB) + db) * 16 + e) * 64 + (threadIdx.x & 63)];
        bool open = true;
        for (int h = hk * rep; open && h < (hk + 1) * rep; ++h)
            for (int i = max(0, k0 - a.right); open && i <= last; ++i) {
                const T *qr = base + (int64_t)i * a.ld + h * HD, *gr = (const T*)a.dout + (start + i) * a.H * HD + h * HD;
                const int64_t at = (int64_t)h * a.R + start + i;
                float w = __builtin_amdgcn_exp2f(dot_half<C>(kv, qr, h2) * c - a.lse[at]);
                if (grad) w *= dot_half<C>(vv, gr, h2) + a.ndelta[at];
                add_half<C>(acc, 1.0f, sees(a, i, key), w, grad ? qr : gr, h2);
                open = !all_nan<C>(acc);
            }
        store_rows<T, HD>(acc, grad ? a.scale : 1.0f, grad ? row : row + a.KV * HD, h2);
    }
}

// dK and dV, the key on the lane: sweeps the queries that see the block's keys, for every query head of the group.
// FAR_FORM: the part that reaches the sinks from queries beyond the window (i > j + left): few keys, all queries of the sequence.  Left to the
// other forms, the block with the sinks would sweep the whole sequence while the rest is long done (backward of 7 sequences of 0 .. 2043 rows,
// one sink: 540 us with, 180 without).  A block takes 32 sinks and every far_parts-th four (head, tile) pairs, and leaves its waves' sum in
// far_ws; with far_parts > 0 the other forms' sums start from there and leave those queries out.
enum { ROW_FORM, SPLIT_FORM, FAR_FORM };
template <typename T, int HD, bool OWN> struct DkvCfg {
    using C = std::conditional_t<OWN, WCfg<T, HD, 32, 1>, WCfg<T, HD, (sizeof(T) == 2 && HD < 128) ? 64 : 32>>;
    static constexpr int STAGE = 2 * C::TILE + 512, STAGES = OWN && C::RB > 256 ? 1 : OWN || STAGE > 20480 ? 2 : 3, BYTES = STAGES * STAGE;      // Q image | dO image | 64 log-sum-exps | 64 row dots
};
template <typename T, int HD, int FORM>
__global__ __launch_bounds__(WT) WAVES_PER_SIMD(WAVES_OWN(WAVES_DKV(sizeof(T) * HD), sizeof(T) * HD, FORM == FAR_FORM || (FORM == SPLIT_FORM && sizeof(T) == 2))) void window_dkv_kernel(WArgs a) {
    constexpr bool OWN = FORM != ROW_FORM, FAR = FORM == FAR_FORM;          // OWN: a wave with tiles of its own
    using D = DkvCfg<T, HD, OWN>;
    using C = typename D::C;
    constexpr int STAGE = D::STAGE, STAGES = D::STAGES, ROWS = OWN ? 32 : WROWS, NC = OWN ? 2 : 1;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    int stream, rblk, part = 0;
    if constexpr (FAR) {
        part = blockIdx.x % a.far_parts;
        rblk = blockIdx.x / a.far_parts % a.far_groups;
        stream = blockIdx.x / (a.far_parts * a.far_groups);
    } else if (!place(a, ROWS, a.NB * a.KV, 1, stream, rblk)) {
        return;
    }
    const int hk = stream % a.KV, b = stream / a.KV;
    int64_t start;
    const int len = seq_rows(a, b, start), kend = FAR ? min(a.sinks, len) : len;        // keys from kend on take no part
    if (rblk * ROWS >= kend) return;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, h2 = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rep = a.H / a.KV;
    const T* base = (const T*)a.qkv + start * a.ld;
    const T *kb_ = base + (a.H + hk) * HD, *vb_ = kb_ + a.KV * HD;
    const int kb0 = rblk * ROWS, k0 = kb0 + (OWN ? 0 : wave * 32), key = k0 + r, klast = min(k0 + 31, kend - 1);
    const int sinks = a.far_parts ? 0 : a.sinks;
    const float c = a.scale * LOG2E;

    typename Frag<T>::V kf[C::FR] = {}, vf[C::FR] = {};
#pragma unroll
    for (int j = 0; j < C::FR; ++j)
        if (key < kend) {
            kf[j] = *reinterpret_cast<const typename Frag<T>::V*>(kb_ + (int64_t)key * a.ld + (2 * j + h2) * (16 / C::ES));
            vf[j] = *reinterpret_cast<const typename Frag<T>::V*>(vb_ + (int64_t)key * a.ld + (2 * j + h2) * (16 / C::ES));
        }
#pragma unroll
    for (int j = 0; j < C::FR; ++j) {
        pin(kf[j]);
        pin(vf[j]);
    }
    f32x16_t dk[C::DB], dv[C::DB];
#pragma unroll
    for (int db = 0; db < C::DB; ++db) dk[db] = dv[db] = splat16(0.f);
    constexpr bool ADD = OWN && C::RB < 256;          // a split block's waves each add up a share of the far parts; else they come folded, to one wave
    const int parts = ADD ? a.far_parts : 1;
    const float* w = a.far_ws + ((int64_t)(b * a.KV + hk) * a.far_groups + k0 / 32) * a.far_parts * (2 * C::DB * 1024);
    if (!FAR && a.far_parts && k0 < min(a.sinks, len) && (ADD || !OWN || wave == 0)) {
        for (int p = ADD ? wave : 0; p < parts; p += 4)
#pragma unroll
            for (int db = 0; db < C::DB; ++db)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    dk[db][e] += w[(int64_t)p * (2 * C::DB * 1024) + (db * 16 + e) * 64 + lane];
                    dv[db][e] += w[(int64_t)p * (2 * C::DB * 1024) + ((C::DB + db) * 16 + e) * 64 + lane];
                }
    }
#pragma unroll
    for (int db = 0; db < C::DB; ++db) asm volatile("" : "+v"(dk[db]), "+v"(dv[db]));

    // queries that see a key of the block: from the first key minus right to the last key plus left, to the end where there are sinks
    const int qlo = FAR ? k0 + a.left + 1 : max(0, kb0 - a.right), qhi = FAR || kb0 < sinks ? len - 1 : min(len - 1, min(kb0 + ROWS, len) - 1 + a.left);
    const int t0 = qlo / C::KT, nt = max(0, qhi / C::KT - t0 + 1);
    // this wave's (head, tile) pairs: w0, w0 + step, ...
    const int step = FAR ? 4 * a.far_parts : OWN ? 4 : 1, w0 = FAR ? part * 4 + wave : OWN ? wave : 0, total = (nt * rep - w0 + step - 1) / step;
    const int64_t gld = (int64_t)a.H * HD;
    const T* gb = (const T*)a.dout + start * gld;
    const float* cb = ((wave & 1) ? a.ndelta : a.lse) + start;         // a shared tile's row constants: the waves alternate, too
    unsigned src[C::NI];
#pragma unroll
    for (int j = 0; j < C::NI; ++j) {       // the waves alternate between the two images: an instruction knows its descriptor
        const int p = OWN ? j : j * 4 + wave;
        src[j] = piece_src<C>(p >= C::NP ? p - C::NP : p, lane, p >= C::NP ? gld : a.ld);
    }
    int ft = OWN && nt ? w0 % nt : 0, fh = hk * rep + (OWN && nt ? w0 / nt : 0);              // the tile and head to fetch next
    auto issue = [&](unsigned char* stage) {
        const int64_t row0 = (int64_t)(t0 + ft) * C::KT, left = len - 1 - row0;
        const __amdgpu_buffer_rsrc_t rq = rows_rsrc(base + fh * HD + row0 * a.ld, (left * a.ld + HD) * C::ES);
        const __amdgpu_buffer_rsrc_t rg = rows_rsrc(gb + fh * HD + row0 * gld, (left * gld + HD) * C::ES);
#pragma unroll
        for (int j = 0; j < C::NI; ++j) {
            const int p = OWN ? j : j * 4 + wave;
            if (p >= C::NP) dma16(rg, stage + p * 1024, src[j]);
            else dma16(rq, stage + p * 1024, src[j]);
        }
        const int64_t crow = (int64_t)fh * a.R + row0;
        if constexpr (OWN) {
            dma4(rows_rsrc(a.lse + start + crow, (left + 1) * 4), stage + 2 * C::TILE, lane * 4);
            dma4(rows_rsrc(a.ndelta + start + crow, (left + 1) * 4), stage + 2 * C::TILE + 256, lane * 4);
        } else {
            dma4(rows_rsrc(cb + crow, (left + 1) * 4), stage + 2 * C::TILE + (wave & 1) * 256, lane * 4);
        }
        for (ft += step; ft >= nt; ft -= nt) ++fh;
    };
    const TrAt<C, (C::RB < 256)> tr(lane);
    const RowAt<C, (C::RB < 256)> rows(lane);
    unsigned char* own = smem + (OWN ? wave * D::BYTES : 0);
    const unsigned lds = lds_u32(own);
    int fill = 0, use = 0, ct = ft;
    for (; fill < STAGES - 1 && fill < total; ++fill) issue(own + fill * STAGE);
    fill = STAGES - 1;
    for (int it = 0; it < total; ++it) {
        if constexpr (STAGES == 1) {
            wait_lds();
            issue(own);
            wait_vm<0>();
        } else {
            tile_ready<(STAGES - 2) * (C::NI + NC), OWN>(it + STAGES - 1 > total);
            if (it + STAGES - 1 < total) issue(own + fill * STAGE);
        }
        fill = fill + 1 == STAGES ? 0 : fill + 1;
        const unsigned ql = lds + use * STAGE, gl = ql + C::TILE;
        use = use + 1 == STAGES ? 0 : use + 1;
        const int q0 = (t0 + ct) * C::KT, q1 = q0 + C::KT - 1;
        for (ct += step; ct >= nt;) ct -= nt;
        if (!FAR && (k0 >= len || q1 < k0 - a.right || (q0 > klast + a.left && k0 >= sinks))) continue;
        const bool whole = FAR ? q1 < len && q0 > klast + a.left && k0 + 31 < kend : q1 < len && q0 >= klast - a.right && (q1 <= k0 + a.left || klast < sinks);
        const int first = FAR ? key + a.left + 1 - q0 : key - a.right - q0;
        const int last = FAR ? (key < kend ? len - 1 - q0 : -1) : (key < sinks ? len - 1 : min(len - 1, key + a.left)) - q0;
        dkv_block<C, 0>(ql, gl, gl + C::TILE, rows, kf, vf, c, whole, first, last, tr, dk, dv, h2);
        if constexpr (C::KB == 2) dkv_block<C, 32>(ql, gl, gl + C::TILE, rows, kf, vf, c, whole, first, last, tr, dk, dv, h2);
    }
    if constexpr (FAR) {
        float* w = a.far_ws + (((int64_t)stream * a.far_groups + rblk) * a.far_parts + part) * (2 * C::DB * 1024) + wave * 256 + lane;
#pragma unroll
        for (int i = 0; i < 2 * C::DB; ++i) {
            float v[4];
            join_block(i < C::DB ? dk[i % C::DB] : dv[i % C::DB], 1.0f, reinterpret_cast<float*>(smem), v, wave, lane);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[i * 1024 + e * 64] = v[e];
        }
        return;
    }
    T* row = (T*)a.dqkv + (start + key) * (a.H + 2 * a.KV) * HD + (a.H + hk) * HD;
    if constexpr (OWN) {
        float* st = reinterpret_cast<float*>(smem);
        __syncthreads();
        const bool bad = any_wave_bad(any_bad<C>(dk) || any_bad<C>(dv), st, wave, lane);
        join_rows<C>(dk, a.scale, st + 512, key < len && !bad, row, wave, lane);
        join_rows<C>(dv, 1.0f, st + 512, key < len && !bad, row + a.KV * HD, wave, lane);
        if (bad && key < len && wave == 0) redo_key<C>(a, base, start, hk, key, k0, len, h2, w, parts, row);
        return;
    }
    if (key < len) {
        if (pair_sum(any_bad<C>(dk) || any_bad<C>(dv) ? 1.0f : 0.f) != 0.f) {
            redo_key<C>(a, base, start, hk, key, k0, len, h2, w, parts, row);
        } else {
            store_rows<T, HD>(dk, a.scale, row, h2);
            store_rows<T, HD>(dv, 1.0f, row + a.KV * HD, h2);
        }
    }
}

// the parts of a group of sinks, added in their order into the first
__global__ __launch_bounds__(WT) void window_far_fold_kernel(float* __restrict__ ws, int parts, int size) {
    const int i = blockIdx.x * WT + threadIdx.x;
    float* w = ws + (int64_t)blockIdx.y * parts * size;
    if (i >= size) return;
    float t = 0.f;
#pragma unroll 4
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
static int64_t grid_of(const WArgs& a, int rows, int heads) {
    const int64_t streams = (int64_t)a.NB * heads;
    return (dealt(a.offsets, (int)streams) ? cdiv(streams, 8) * 8 : streams) * cdiv(a.L, rows);
}
// Split form or row form, by the 128-row blocks that the row form would have, in eighths of the compute units.  Below the limits the split form
// was faster, above them the row form (1024 rows, 8 .. 80 heads, windows 64 and 512, forward in us, split / row: hd 32 10.5 / 12.0 at 256 blocks
// and 15.4 / 15.7 at 448; hd 64 9.2 / 13.8 at 128, 13.8 / 14.2 at 192, 26.1 / 19.2 at 448; hd 128 10.1 / 17.1 at 64, 18.2 / 18.0 at 128; float32 hd 16
// 40.5 / 46.9 at 896, hd 32 29.5 / 35.5 at 256, hd 64 34.8 / 57.2 at 128, 61.3 / 58.4 at 256, hd 128 17 / 55 at 48, 168 / 149 at 256).  dK/dV has a longer sweep per block, over every head of
// a group: its limits lie higher (dK/dV + dQ, 4 heads a group, window 256: hd 128 44.6 / 95.7 at 64 blocks, 120 / 131 at 160; hd 64 55 / 69 at 160).
// A window open to one side leaves blocks with long and with short sweeps, and the launch waits for the longest, which the split form cuts in four:
// higher limits from 1024 and from 2048 keys on (causal, 4096 rows: hd 32 47 / 68 at 512 blocks, 71 / 89 at 768; hd 64 36 / 65 at 256, 97 / 106 at
// 768; hd 128 69 / 79 at 256, 136 / 113 at 512; float32 hd 32 165 / 309 at 512, 247 / 442 at 768, hd 128 325 / 561 at 256, 629 / 644 at 512, 952 /
// 1201 at 768, 1243 / 1215 at 1024; 1536 rows: 121 / 224 at 192, 318 / 431 at 576; with a window of 1024 as for the others.  The
// whole backward pass, dK/dV split / row: hd 32 114 / 144 at 512, hd 64 174 / 203, hd 128 214 / 290 at 256, 4 heads a group 599 / 959; float32 hd
// 64 1124 / 1476 at 512, hd 128 1137 / 1968 at 256, 3436 / 4209 at 768, 1536 rows 407 / 754 at 192, 1137 / 1512 at 576).
template <typename T, int HD> struct SplitUpTo {
    static constexpr int RB = HD * sizeof(T);
    static constexpr bool BF = sizeof(T) == 2;
    static int rows(int sweep) {
        constexpr int R[3] = {BF ? (RB <= 64 ? 10 : RB <= 128 ? 4 : 3) : (RB <= 64 ? 28 : RB <= 128 ? 10 : RB <= 256 ? 5 : 4),
                              BF ? (RB <= 64 ? 16 : RB <= 128 ? 8 : 4) : (RB <= 64 ? 28 : 24), BF ? (RB <= 128 ? 24 : 8) : (RB <= 64 ? 28 : 24)};
        return R[sweep];
    }
    static int keys(int sweep) {
        constexpr int K[3] = {BF ? (RB <= 64 ? 12 : RB <= 128 ? 8 : 5) : (RB <= 128 ? 20 : RB <= 256 ? 12 : 7), BF ? (RB <= 64 ? 24 : RB <= 128 ? 12 : 10) : (RB <= 128 ? 40 : 24),
                              BF ? (RB <= 64 ? 24 : RB <= 128 ? 16 : 20) : (RB <= 128 ? 40 : 24)};
        return K[sweep];
    }
};
// 0: sweeps of about one length, or short ones; 1, 2: a window open to one side with sweeps of up to 1024, 2048 keys and more
static int sweep_class(const WArgs& a) {
    const int wide = a.left > a.right ? a.left : a.right, other = a.left > a.right ? a.right : a.left;
    if (2 * wide < a.L || 4 * other >= a.L) return 0;
    const int keys = wide + other + WROWS < a.L ? wide + other + WROWS : a.L;
    return keys >= 2048 ? 2 : keys >= 1024 ? 1 : 0;
}
// (a sweep of one tile has nothing to split: 1 x 32 rows, 8 heads, forward 4.4 us by rows and 4.6 split at hd 32, 8.7 and 11.0 in float32 at hd 128)
static bool few_blocks(const WArgs& a, int heads, int eighths) {
    if ((int64_t)(a.H / heads) * cdiv(a.L, 32) == 1) return false;
    const int64_t blocks = (a.offsets ? cdiv(a.R, WROWS) : (int64_t)a.NB * cdiv(a.L, WROWS)) * (int64_t)heads;
    return blocks * 8 <= (int64_t)eighths * star_num_cus();
}
template <typename T, int HD, bool SPLIT> static int launch_fwd(const WArgs& a, hipStream_t s) {
    using Ring = KvRing<RowCfg<T, HD, SPLIT>>;
    constexpr int LDS = SPLIT ? 4 * Ring::BYTES : Ring::BYTES;
    return launch<window_fwd_kernel<T, HD, SPLIT>>("star_attn_window_fwd", grid_of(a, SPLIT ? 32 : WROWS, a.H) + a.rest_blocks, SPLIT && LDS < 18432 ? 18432 : LDS, a, s);
}
template <typename T, int HD, bool SPLIT> static int launch_dq(const WArgs& a, hipStream_t s) {
    using Ring = KvRing<RowCfg<T, HD, SPLIT>>;
    constexpr int LDS = SPLIT ? 4 * Ring::BYTES : Ring::BYTES;
    return launch<window_dq_kernel<T, HD, SPLIT>>("star_attn_window_bwd", grid_of(a, SPLIT ? 32 : WROWS, a.H) + a.rest_blocks, SPLIT && LDS < 18432 ? 18432 : LDS, a, s);
}
template <typename T, int HD, int FORM> static int launch_dkv(const WArgs& a, hipStream_t s) {
    constexpr bool OWN = FORM != ROW_FORM;
    using D = DkvCfg<T, HD, OWN>;
    constexpr int LDS = OWN ? 4 * D::BYTES : D::BYTES;
    const int64_t blocks = FORM == FAR_FORM ? (int64_t)a.NB * a.KV * a.far_groups * a.far_parts : grid_of(a, OWN ? 32 : WROWS, a.KV);
    return launch<window_dkv_kernel<T, HD, FORM>>("star_attn_window_bwd", blocks, OWN && LDS < 18432 ? 18432 : LDS, a, s);
}
// the hardware counts a launch's threads in 32 bits: checked before the first launch of a call
static bool grid_fits(const WArgs& a, bool split, int heads) { return (grid_of(a, split ? 32 : WROWS, heads) + a.rest_blocks) * WT < (1ll << 32); }
template <typename T, int HD> static int run_fwd(const WArgs& a, hipStream_t s) {
    using S = SplitUpTo<T, HD>;
    const bool split = few_blocks(a, a.H, S::rows(sweep_class(a)));
    STAR_CHECK(grid_fits(a, split, a.H), "star_attn_window_fwd: NB, H, L too large for the grid");
    if (split) return launch_fwd<T, HD, true>(a, s);
    return launch_fwd<T, HD, false>(a, s);
}
template <typename T, int HD> static int run_dq(const WArgs& a, hipStream_t s) {
    using S = SplitUpTo<T, HD>;
    if (few_blocks(a, a.H, S::rows(sweep_class(a)))) return launch_dq<T, HD, true>(a, s);
    return launch_dq<T, HD, false>(a, s);
}
template <typename T, int HD> static int run_dkv(const WArgs& a, hipStream_t s) {
    using S = SplitUpTo<T, HD>;
    if (few_blocks(a, a.KV, S::keys(sweep_class(a)))) return launch_dkv<T, HD, SPLIT_FORM>(a, s);
    return launch_dkv<T, HD, ROW_FORM>(a, s);
}
template <typename T, int HD> static int run_bwd(const WArgs& first, hipStream_t s) {
    const char* who = "star_attn_window_bwd";
    using S = SplitUpTo<T, HD>;
    const int sweep = sweep_class(first);
    STAR_CHECK(grid_fits(first, few_blocks(first, first.H, S::rows(sweep)), first.H) && grid_fits(first, few_blocks(first, first.KV, S::keys(sweep)), first.KV),
               "%s: NB, H, L too large for the grid", who);
    int rc = run_dq<T, HD>(first, s);
    if (rc) return rc;
    WArgs a = first;
    a.rest_blocks = 0;
    if (a.far_parts) {
        if ((rc = launch_dkv<T, HD, FAR_FORM>(a, s))) return rc;
        // the split form adds the parts up itself where a row is under 256 bytes (7 sequences of 0 .. 2043 rows, 16 heads on 4 of 64: 122 us against
        // 128; 128-wide heads have too few registers to keep the loads in flight: 102 against 48)
        if (a.far_parts > 1 && !(HD * sizeof(T) < 256 && few_blocks(a, a.KV, S::keys(sweep)))) {
            const int size = 2 * WCfg<T, HD>::DB * 1024;
            hipLaunchKernelGGL(window_far_fold_kernel, dim3(size / WT, a.NB * a.KV * a.far_groups), dim3(WT), 0, s, a.far_ws, a.far_parts, size);
            STAR_LAUNCH_CHECK(who);
        }
    }
    return run_dkv<T, HD>(a, s);
}

// How the far queries of the sinks are cut: about two blocks of four waves per compute unit in all, no more than 16 parts to add up, and at least
// two 32-query tiles for a wave.  No parts with under 24 tiles per key head, which the sinks' own block takes in the time of the other launches
// (without parts / with: float32, 500 rows, 8 heads of 64, 13 tiles: 49 / 75 us; 4 x 700 rows, 16 heads, 18 tiles: 212 / 226; 2 x 1000 rows, 12
// heads of 32, 24 tiles: 91.7 / 88.5; 4 x 1000 rows, 16 heads of 64, 29 tiles: 390 / 263; bf16, 20 x 900 rows, 12 heads of 64, 27 tiles: 192 / 169).
// Over 256 sinks: none where their own blocks are enough to fill the chip or a third of all keys, so that no few of them are waited for (backward,
// without / with: 1 x 8192 rows, 4 heads on 1, 257 sinks, 9 lists of 32: bf16 of 64 288 / 87 us, of 128 419 / 118, float32 of 128 2519 / 535; 1 x 4096, 8
// heads, 300 sinks, 80 lists: 75 / 82, 244 / 140, 1366 / 553; 1 x 4096, 8 heads, 1000 sinks, 256 lists: 89 / 101, 262 / 175, 1496 / 832; 8 x 2048, 16
// heads, 300 sinks, 1280 lists: 250 / 259, 491 / 511, 3296 / 2879; 2 x 1024, 4 heads, 500 sinks, 128 lists: 30 / 37, 40 / 60, 144 / 149).
static void far_plan(int NB, int L, int H, int KV, int left, int sinks, int row_bytes, int& groups, int& parts) {
    groups = parts = 0;
    sinks = sinks < L ? sinks : L;
    if (sinks <= 0 || left >= L - 1) return;
    const int64_t lists = (int64_t)NB * KV * cdiv(sinks, 32), tiles = (int64_t)(H / KV) * cdiv(L - left - 1, 32), cus = star_num_cus();
    if (lists > 65535 || tiles < 24) return;
    if (sinks > 256 && (3 * (int64_t)sinks > L || 2 * lists > (row_bytes < 256 ? 1 : 4) * cus)) return;
    groups = cdiv(sinks, 32);
    int64_t p = cdiv(2 * cus, lists);
    if (p > tiles / 8) p = tiles / 8;
    parts = p < 1 ? 1 : p > 16 ? 16 : (int)p;
}

static int longest(int L, int64_t R) { return L < R ? L : R < 1 ? 1 : (int)R; }
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
    STAR_CHECK((int64_t)cdiv(longest(g->L, g->R), 32) * ((int64_t)g->H * g->NB + 7) < (1ll << 31) - 1024, "%s: NB, H, L too large for the grid", who);
    // a bound over L says the same as L (what is left cannot overflow in i + right and i - left), and L over all rows the same as R: no blocks for those
    const int L = longest(g->L, g->R);
    a = WArgs{g->qkv, g->offsets, g->out, g->lse, nullptr, nullptr, nullptr, nullptr, g->ld, g->R, g->NB, L, g->H, g->KV,
              g->left < L ? g->left : L, g->right < L ? g->right : L, g->sinks < L ? g->sinks : L, g->scale, 0, 0, 0};
    return 0;
}
// a block per 256 KiB of a matrix of R rows that is to be zeroed outside the sequences (most of it is inside as a rule): a fill of the whole
// costs a launch and all its bytes
static int rest_blocks(const StarAttnWindow* g, int64_t width) {
    if (!g->offsets || !g->zero_rest) return 0;
    const int64_t n = g->R * width * (g->dt == STAR_BF16 ? 2 : 4) >> 18;
    return n < 1 ? 1 : n > 512 ? 512 : (int)n;
}

#define BY_HD(F, T)                                                                         \
    (g->hd == 16 ? F<T, 16>(a, s) : g->hd == 32 ? F<T, 32>(a, s) : g->hd == 64 ? F<T, 64>(a, s) : F<T, 128>(a, s))

extern "C" int star_attn_window_fwd(const StarAttnWindow* g, void* stream) {
    WArgs a;
    if (int rc = window_args("star_attn_window_fwd", g, a)) return rc;
    // blocks read rows that others may have written results over already.  (A single row in place: a head's block alone reads its query.)
    const int64_t es = g->dt == STAR_BF16 ? 2 : 4, orow = (int64_t)g->H * g->hd * es, lse = (int64_t)g->H * g->R * 4;
    const int64_t row = ((int64_t)g->H + 2 * (int64_t)g->KV) * g->hd * es;
    STAR_CHECK((g->R == 1 && g->out == g->qkv) || !star_meets(g->out, g->R * orow, g->qkv, g->R, g->ld * es, row), "star_attn_window_fwd: out overlaps qkv");
    STAR_CHECK(!star_meets(g->lse, lse, g->qkv, g->R, g->ld * es, row) && !star_meets(g->lse, lse, g->out, g->R * orow), "star_attn_window_fwd: lse overlaps qkv or out");
    a.rest_blocks = rest_blocks(g, (int64_t)g->H * g->hd);
    hipStream_t s = (hipStream_t)stream;
    return g->dt == STAR_BF16 ? BY_HD(run_fwd, bf16_t) : BY_HD(run_fwd, float);
}

extern "C" int64_t star_attn_window_bwd_ws(int64_t R, int NB, int L, int H, int KV, int hd, int left, int sinks, int dt) {
    if (R < 0 || NB <= 0 || L <= 0 || H <= 0 || KV <= 0 || H % KV || hd <= 0 || left < 0 || sinks < 0) return 0;
    int groups, parts;
    far_plan(NB, longest(L, R), H, KV, left, sinks, hd * (dt == STAR_BF16 ? 2 : 4), groups, parts);
    return (H * R + 63) / 64 * 64 + (int64_t)NB * KV * groups * parts * 2 * 32 * (hd < 32 ? 32 : hd);
}

extern "C" int star_attn_window_bwd(const StarAttnWindow* g, void* stream) {
    WArgs a;
    if (int rc = window_args("star_attn_window_bwd", g, a)) return rc;
    STAR_CHECK(g->lse && g->dout && g->dqkv && g->ws, "star_attn_window_bwd: null pointer");
    STAR_CHECK((uintptr_t)g->dout % 16 == 0 && (uintptr_t)g->dqkv % 16 == 0, "star_attn_window_bwd: dout and dqkv must be 16-byte aligned");
    // the dK/dV launches read what the dQ launch has read before them
    const int64_t es = g->dt == STAR_BF16 ? 2 : 4, orow = (int64_t)g->H * g->hd * es, lse = (int64_t)g->H * g->R * 4;
    const int64_t row = ((int64_t)g->H + 2 * (int64_t)g->KV) * g->hd * es;
    const int64_t ws = star_attn_window_bwd_ws(g->R, g->NB, g->L, g->H, g->KV, g->hd, g->left, g->sinks, g->dt) * 4;
    auto meets = [&](const void* p, int64_t n) {
        return star_meets(p, n, g->qkv, g->R, g->ld * es, row) || star_meets(p, n, g->out, g->R * orow) || star_meets(p, n, g->dout, g->R * orow) || star_meets(p, n, g->lse, lse);
    };
    STAR_CHECK(!meets(g->dqkv, g->R * row), "star_attn_window_bwd: dqkv overlaps qkv, out, dout or lse");
    STAR_CHECK(!meets(g->ws, ws) && !star_meets(g->ws, ws, g->dqkv, g->R * row), "star_attn_window_bwd: ws overlaps another operand");
    a.dout = g->dout;
    a.dqkv = g->dqkv;
    a.ndelta = g->ws;
    a.rest_blocks = rest_blocks(g, (int64_t)(g->H + 2 * g->KV) * g->hd);
    far_plan(g->NB, a.L, g->H, g->KV, g->left, g->sinks, g->hd * (int)es, a.far_groups, a.far_parts);
    a.far_ws = g->ws + (g->H * g->R + 63) / 64 * 64;
    hipStream_t s = (hipStream_t)stream;
    return g->dt == STAR_BF16 ? BY_HD(run_bwd, bf16_t) : BY_HD(run_bwd, float);
}
