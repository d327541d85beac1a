// Rotary positions with several axes (time, row, column of a token ...), forward and backward.
//
// Pair i of a head turns by the angle theta_i = pos[axis(i)] * f_i:  y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin; the backward pass is the
// rotation by -theta.  A pair is (i, i + n) of the first 2 n elements of the head, or (2 i, 2 i + 1).
// Memory-bound: every element read and written once, ~3 flop per element.  A block takes a few rows: its threads first compute each
// (row, pair)'s cosine and sine once into LDS, then stream through the rows with 16-byte accesses, every head reading the same table.
// Angles are formed in revolutions in float64 (a float32 product would lose the fraction of far positions); the fraction left after
// dropping whole revolutions is exact enough in float32.
// Measured: 40960 rows of 36 heads of 32 in bf16, 24 of them turned (189 MB read and written): 45 us = 4.2 TB/s (a copy: 4.7).
#include "common.h"

#define RT 256
#define MAX_ROWS 8
#define MAX_PAIRS 64

struct RopeArgs {
    const void* x;
    void* y;
    const int32_t* pos;
    int64_t x_ld, y_ld, pos_ld;
    int R, W, rot, hd, rows;       // rows: rows of a block
    float sign;
    StarRope f;
};

template <typename T> __device__ __forceinline__ void ld8(const T* p, float (&v)[8]) {
    float a[4], b[4];
    ld4(p, a);
    ld4(p + 4, b);
#pragma unroll
    for (int k = 0; k < 4; ++k) { v[k] = a[k]; v[4 + k] = b[k]; }
}
template <typename T> __device__ __forceinline__ void st8(T* p, const float (&v)[8]) {
    const float a[4] = {v[0], v[1], v[2], v[3]}, b[4] = {v[4], v[5], v[6], v[7]};
    st4(p, a);
    st4(p + 4, b);
}

template <typename T>
__global__ __launch_bounds__(RT) void rope_kernel(RopeArgs a) {
    __shared__ float cs[MAX_ROWS * MAX_PAIRS], sn[MAX_ROWS * MAX_PAIRS];
    const int row0 = blockIdx.x * a.rows, nrow = min(a.rows, a.R - row0), n = a.f.pairs;
    for (int i = threadIdx.x; i < nrow * n; i += RT) {
        const int row = i / n, k = i % n;
        const double rev = (double)a.pos[a.f.axis[k] * a.pos_ld + row0 + row] * a.f.rev[k];
        const float half = 2.0f * (float)(rev - rint(rev));          // half revolutions in [-1, 1]
        sincospif(half, &sn[i], &cs[i]);
        sn[i] *= a.sign;
    }
    __syncthreads();
    const int nc = n / 8, per = a.hd / 8;                    // rotating items (8 pairs) and 8-element chunks of a head
    const int nrot = a.rot * nc;
    // out of place: the elements that do not turn -- the rest of the rotated heads and the columns behind them -- are copied
    const int tail = per - 2 * nc, ncopy = a.x == a.y ? 0 : a.rot * tail + (a.W - a.rot * a.hd) / 8;
    const int items = nrot + ncopy;
    for (int i = threadIdx.x; i < nrow * items; i += RT) {
        const int row = i / items, it = i % items;
        const T* x = (const T*)a.x + (int64_t)(row0 + row) * a.x_ld;
        T* y = (T*)a.y + (int64_t)(row0 + row) * a.y_ld;
        if (it < nrot) {
            const int head = it / nc, k = (it % nc) * 8;
            const float *c = cs + row * n + k, *s = sn + row * n + k;
            const int o1 = head * a.hd + (a.f.interleaved ? 2 * k : k), o2 = o1 + (a.f.interleaved ? 8 : n);
            float u[8], v[8];
            ld8(x + o1, u);
            ld8(x + o2, v);
            if (a.f.interleaved) {
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const float p = u[j], q = v[j];
                    u[j] = p * c[j / 2] - u[j + 1] * s[j / 2];
                    u[j + 1] = u[j + 1] * c[j / 2] + p * s[j / 2];
                    v[j] = q * c[4 + j / 2] - v[j + 1] * s[4 + j / 2];
                    v[j + 1] = v[j + 1] * c[4 + j / 2] + q * s[4 + j / 2];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float p = u[j];
                    u[j] = p * c[j] - v[j] * s[j];
                    v[j] = v[j] * c[j] + p * s[j];
                }
            }
            st8(y + o1, u);
            st8(y + o2, v);
        } else {
            const int k = it - nrot, nt = a.rot * tail;
            const int o = k < nt ? (k / tail) * a.hd + 2 * n + (k % tail) * 8 : a.rot * a.hd + (k - nt) * 8;
            float u[8];
            ld8(x + o, u);
            st8(y + o, u);
        }
    }
}

extern "C" int star_rope(const void* x, int64_t x_ld, void* y, int64_t y_ld, const int32_t* pos, int64_t pos_ld, const StarRope* h_rope, int R,
                         int W, int rot_heads, int hd, int inverse, int dt, void* stream) {
    STAR_CHECK(x && y && pos && h_rope, "star_rope: null pointer");
    STAR_CHECK(dt == STAR_BF16 || dt == STAR_F32, "star_rope: dtype %d is neither STAR_BF16 nor STAR_F32", dt);
    STAR_CHECK(R >= 0 && rot_heads > 0 && hd > 0 && hd % 16 == 0 && hd <= 65536 && W % 8 == 0 && W / hd >= rot_heads,
               "star_rope: bad shape R=%d W=%d, %d heads of %d", R, W, rot_heads, hd);
    const int n = h_rope->pairs;
    STAR_CHECK(n > 0 && n <= MAX_PAIRS && n % 8 == 0 && 2 * n <= hd, "star_rope: %d pairs in heads of %d (a multiple of 8, at most %d)", n, hd, MAX_PAIRS);
    STAR_CHECK(h_rope->axes > 0, "star_rope: no position axes");
    for (int i = 0; i < n; ++i) STAR_CHECK(h_rope->axis[i] < h_rope->axes, "star_rope: pair %d turns by axis %d of %d", i, h_rope->axis[i], h_rope->axes);
    const int es = dt == STAR_BF16 ? 2 : 4;
    STAR_CHECK(x_ld >= W && y_ld >= W && x_ld * es % 16 == 0 && y_ld * es % 16 == 0 && (uintptr_t)x % 16 == 0 && (uintptr_t)y % 16 == 0,
               "star_rope: rows must hold %d elements and be 16-byte aligned", W);
    STAR_CHECK(pos_ld >= R, "star_rope: position rows of %lld for %d tokens", (long long)pos_ld, R);
    STAR_CHECK(x != y || x_ld == y_ld, "star_rope: in place with two row strides");
    // x and y may be column ranges of one matrix, but no element of both: a thread's row may be read by another after it is written
    const int64_t gap = ((intptr_t)y - (intptr_t)x) / es, before = gap < 0 ? -gap : gap, low_ld = gap < 0 ? y_ld : x_ld;
    if (gap && R > 0 && before < (R - 1) * low_ld + W) {
        const int64_t off = before % low_ld;
        STAR_CHECK(x_ld == y_ld && off >= W && low_ld - off >= W, "star_rope: x and y overlap");
    }
    if (R == 0) return 0;
    // a few rows per block so that the angle pass fills its threads; single rows while there are fewer blocks than compute units
    int rows = MAX_ROWS;
    while (rows > 1 && cdiv(R, rows) < 2 * star_num_cus()) rows /= 2;
    // the hardware counts a launch's threads in 32 bits: 2^26 rows at a time
    const int most = 1 << 26;
    hipStream_t s = (hipStream_t)stream;
    for (int64_t r0 = 0; r0 < R; r0 += most) {
        const int part = R - r0 < most ? (int)(R - r0) : most;
        const RopeArgs a = {(const char*)x + r0 * x_ld * es, (char*)y + r0 * y_ld * es, pos + r0, x_ld, y_ld, pos_ld, part, W, rot_heads, hd, rows, inverse ? -1.0f : 1.0f, *h_rope};
        if (dt == STAR_BF16) hipLaunchKernelGGL(rope_kernel<bf16_t>, dim3(cdiv(part, rows)), dim3(RT), 0, s, a);
        else hipLaunchKernelGGL(rope_kernel<float>, dim3(cdiv(part, rows)), dim3(RT), 0, s, a);
        STAR_LAUNCH_CHECK("star_rope");
    }
    return 0;
}
