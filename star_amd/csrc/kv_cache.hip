// The rolling key/value cache of sliding-window attention with sinks, and the attention of one new token per sequence over it.
//
// cache [2 (keys, values), NB, KV, cap, hd]: the token at position p lies in slot p for p < sinks, else in slot
// sinks + (p - sinks) % (cap - sinks), so the ring behind the sinks holds the newest cap - sinks tokens (cap >= the longest sequence: an
// ordinary cache).  lengths [NB] counts a sequence's tokens including the new ones; 0 marks an idle entry.
//
// Both kernels are bound by the bytes of the cache rows they touch: 16 prompts of 301 .. 6000 rows, 8 heads of 128 in bf16: 70 us = 5.2 TB/s;
// a step of 64 sequences of 3000 .. 20000 tokens (8196 slots), 32 heads on 8 of 128: 359 us = 5.4 TB/s (a copy: 4.7, reads only need no turn-around).  Small calls
// are bound by latency and by what one compute unit reads: 5 sequences, 12 heads of 64, up to 1040 tokens: 9.9 us in one launch.
#include "common.h"

#define KT_ 256
#define LOG2E 1.4426950408889634f

struct AppendArgs {
    const void* qkv;
    const int64_t* offsets;
    void* cache;
    const int32_t* lengths;
    int64_t ld, R;
    int NB, L, H, KV, hd, cap, sinks;
};

template <int ES>
__global__ __launch_bounds__(KT_) void kv_append_kernel(AppendArgs a) {
    const int per = a.hd * ES / 16, cols = a.KV * per;            // 16-byte chunks of a head's row, of a token's keys
    const int b = blockIdx.y;
    int64_t start = (int64_t)b * a.L, n = a.L;
    if (a.offsets) {        // whatever the device-side offsets hold, rows stay inside [0, R)
        int64_t s = a.offsets[b], e = a.offsets[b + 1];
        s = s < 0 ? 0 : (s > a.R ? a.R : s);
        e = e < s ? s : (e > a.R ? a.R : e);
        start = s;
        n = e - s > a.L ? a.L : e - s;
    }
    const int64_t total = a.lengths[b], first = total - n;
    const int ring = a.cap - a.sinks;
    const int64_t end = n * 2 * cols;
    for (int64_t i = (int64_t)blockIdx.x * KT_ + threadIdx.x; i < end; i += (int64_t)gridDim.x * KT_) {
        const int64_t t = i / (2 * cols);
        const int k = (int)(i % (2 * cols)), half = k / cols, head = k % cols / per, ch = k % per;
        const int64_t p = first + t;
        if (p < 0 || (p >= a.sinks && p < total - ring)) continue;      // older than the ring holds
        const int64_t slot = p < a.sinks ? p : a.sinks + (p - a.sinks) % ring;
        const char* src = (const char*)a.qkv + ((start + t) * a.ld + (int64_t)(a.H + half * a.KV + head) * a.hd) * ES + ch * 16;
        char* dst = (char*)a.cache + ((((int64_t)half * a.NB + b) * a.KV + head) * a.cap + slot) * a.hd * ES + ch * 16;
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
    }
}

// ------------------------------------------------------------------------------------------------------
struct StepArgs {
    const void* qkv;
    void* cache;
    const int32_t* lengths;
    const int32_t* pos;
    void* out;
    float* ws;               // [NB * H, splits, hd + 2]: unnormalised rows, maximum, sum
    int64_t ld, pos_ld;
    int NB, H, KV, cap, left, sinks, splits, chunks;
    float scale;
    StarRope f;              // pairs = 0: no rotation
};

// sum over the LPR lanes that share a row, in every one of them (DPP exchanges: no LDS round trip)
template <int CTRL> __device__ __forceinline__ float dpp_add(float v) {
    return v + __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float swap16_add(float v) {          // + lane ^ 16
    typedef __attribute__((ext_vector_type(2))) unsigned u2;
    const u2 x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}
template <int LPR> __device__ __forceinline__ float lane_sum(float v) {
    if constexpr (LPR >= 2) v = dpp_add<0xB1>(v);        // quad_perm 1,0,3,2
    if constexpr (LPR >= 4) v = dpp_add<0x4E>(v);        // quad_perm 2,3,0,1
    if constexpr (LPR >= 8) v = dpp_add<0x141>(v);       // row_half_mirror: the other quad of eight
    if constexpr (LPR >= 16) v = dpp_add<0x140>(v);      // row_mirror: the other eight of sixteen
    if constexpr (LPR >= 32) v = swap16_add(v);
    return v;
}
// op over the 64 / LPR lanes that hold the same chunk of other rows (lane % LPR), in every one of them: rotations within 16 lanes, then swaps
// (a shuffle through LDS costs several times as much, and a block has 16 waves and up to 8 heads to join)
template <int CTRL> __device__ __forceinline__ float dpp_get(float v) { return __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(v), CTRL, 0xf, 0xf, true)); }
template <int LPR, class OP> __device__ __forceinline__ float over_rows(float v, OP op) {
    typedef __attribute__((ext_vector_type(2))) unsigned u2;
    if constexpr (LPR <= 8) v = op(v, dpp_get<0x128>(v));          // row_ror 8, 4, 2
    if constexpr (LPR <= 4) v = op(v, dpp_get<0x124>(v));
    if constexpr (LPR <= 2) v = op(v, dpp_get<0x122>(v));
    if constexpr (LPR <= 16) {
        const u2 x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = op(__uint_as_float(x[0]), __uint_as_float(x[1]));
    }
    const u2 x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return op(__uint_as_float(x[0]), __uint_as_float(x[1]));
}
template <typename T> __device__ __forceinline__ void unpack(uint4 w, float (&v)[16 / sizeof(T)]) {
    const unsigned x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (sizeof(T) == 2) {
            v[2 * k] = __uint_as_float(x[k] << 16);
            v[2 * k + 1] = __uint_as_float(x[k] & 0xffff0000u);
        } else {
            v[k] = __uint_as_float(x[k]);
        }
    }
}

// the tokens that a query at position p = len - 1 sees, numbered 0 .. vis - 1: the sinks in front of the window, then the window
struct Seen {
    int ws, nsv, vis, w1, base, sinks, ring;
    __device__ __forceinline__ Seen(int len, int left, int sinks_, int cap) {
        const int p = len - 1;
        sinks = sinks_;
        ring = cap - sinks_;
        ws = max(0, p - left);
        nsv = min(sinks, ws);
        vis = len > 0 ? nsv + p - ws + 1 : 0;
        w1 = max(ws, sinks);
        base = (w1 - sinks) % ring;
    }
    __device__ __forceinline__ int slot(int v) const {
        const int pos = v < nsv ? v : ws + v - nsv;
        if (pos < sinks) return pos;
        const int s = base + pos - w1;                   // the window is not longer than the ring: one wrap at most
        return sinks + (s >= ring ? s - ring : s);
    }
};

// One block: G query heads of one key head of one sequence over one split of the visible tokens.  A row's 16-byte chunks lie on LPR lanes;
// every group of LPR lanes walks its own rows, U at a time, with its own running maximum and sum (no exchange but the dot products'); the
// groups are joined once at the end.  The split that owns the newest token puts it into the cache first, and reads it from there.
template <typename T, int HD, int G, int NT>
__global__ __launch_bounds__(NT) void step_kernel(StepArgs a) {
    constexpr int ES = sizeof(T), E = 16 / ES, LPR = HD / E, RPB = NT / LPR, U = 4, NW = NT / 64;
    __shared__ float sq[G][HD];
    __shared__ float so[NW][G][HD];
    __shared__ float sm[NW][G], sl[NW][G];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // blocks go to the 8 XCDs in turn: those that read the same rows for other query heads are 8 apart, in one L2
    const int gc = (blockIdx.x >> 3) % a.chunks, unit = (blockIdx.x >> 3) / a.chunks * 8 + (blockIdx.x & 7);
    const int split = unit % a.splits, hk = unit / a.splits % a.KV, b = unit / (a.splits * a.KV);
    if (b >= a.NB) return;
    const int rep = a.H / a.KV, h0 = hk * rep + gc * G, ng = min(G, rep - gc * G);
    const int len = max(0, a.lengths[b]);
    const Seen seen(len, a.left, a.sinks, a.cap);
    constexpr int ROUND = RPB * U;
    const int per = ((seen.vis + a.splits - 1) / a.splits + ROUND - 1) / ROUND * ROUND;          // whole rounds
    const int64_t begin = (int64_t)split * per;
    const int v0 = (int)(begin < seen.vis ? begin : seen.vis), v1 = min(seen.vis, v0 + per);
    const bool owner = v1 == seen.vis && v0 < v1;
    const T* row = (const T*)a.qkv + b * a.ld;
    T* kc = (T*)a.cache + ((int64_t)b * a.KV + hk) * a.cap * HD;
    T* vc = kc + (int64_t)a.NB * a.KV * a.cap * HD;

    // rotate the query heads (and, in the owner, the key) once: items = pairs of the rotated part, then single elements of the rest
    const int n = a.f.pairs, rest = HD - 2 * n, items = n + rest;
    const int newest = owner ? seen.slot(seen.vis - 1) : 0;
    for (int i = tid; i < (ng + (owner ? 1 : 0)) * items; i += NT) {
        const int g = i / items, k = i % items;
        const T* src = row + (g < ng ? h0 + g : a.H + hk) * HD;
        T* kd = kc + (int64_t)newest * HD;
        if (k < n) {
            const int i1 = a.f.interleaved ? 2 * k : k, i2 = a.f.interleaved ? 2 * k + 1 : k + n;
            const double rev = (double)a.pos[a.f.axis[k] * a.pos_ld + b] * a.f.rev[k];
            float sn, cs;
            sincospif(2.0f * (float)(rev - rint(rev)), &sn, &cs);
            const float x1 = Act<T>::ld(src + i1), x2 = Act<T>::ld(src + i2);
            const float y1 = x1 * cs - x2 * sn, y2 = x2 * cs + x1 * sn;
            if (g < ng) {
                sq[g][i1] = y1 * a.scale;
                sq[g][i2] = y2 * a.scale;
            } else {
                Act<T>::st(kd + i1, y1);
                Act<T>::st(kd + i2, y2);
            }
        } else {
            const int d = n + k;
            if (g < ng) sq[g][d] = Act<T>::ld(src + d) * a.scale;
            else kd[d] = src[d];
        }
    }
    if (owner)
        for (int d = tid; d < HD; d += NT) vc[(int64_t)newest * HD + d] = row[(a.H + a.KV + hk) * HD + d];
    __syncthreads();

    const int grp = tid / LPR, ch = tid % LPR;
    float q[G][E], o[G][E], m[G], l[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        m[g] = -INFINITY;
        l[g] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            q[g][e] = g < ng ? sq[g][ch * E + e] : 0.f;
            o[g][e] = 0.f;
        }
    }
    for (int vb = v0; vb < v1; vb += ROUND) {
        uint4 kw[U], vw[U];
        bool ok[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int v = vb + u * RPB + grp;
            ok[u] = v < v1;
            kw[u] = vw[u] = make_uint4(0, 0, 0, 0);
            if (ok[u]) {
                const int64_t at = (int64_t)seen.slot(v) * HD + ch * E;
                kw[u] = *reinterpret_cast<const uint4*>(kc + at);
                vw[u] = *reinterpret_cast<const uint4*>(vc + at);
            }
        }
        float s[U][G];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float k[E];
            unpack<T>(kw[u], k);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float d = 0.f;
#pragma unroll
                for (int e = 0; e < E; ++e) d = __builtin_fmaf(q[g][e], k[e], d);
                d = lane_sum<LPR>(d);
                s[u][g] = ok[u] ? d : -INFINITY;
            }
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            float mn = m[g];
#pragma unroll
            for (int u = 0; u < U; ++u) mn = fmaxf(mn, s[u][g]);
            const float ref = mn == -INFINITY ? 0.f : mn;            // a group without a row in this pass: every weight 0
            const float alpha = __builtin_amdgcn_exp2f(m[g] - ref);
            m[g] = mn;
            l[g] *= alpha;
#pragma unroll
            for (int e = 0; e < E; ++e) o[g][e] *= alpha;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                s[u][g] = __builtin_amdgcn_exp2f(s[u][g] - ref);
                l[g] += s[u][g];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float v[E];
            unpack<T>(vw[u], v);
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int e = 0; e < E; ++e) o[g][e] = __builtin_fmaf(s[u][g], v[e], o[g][e]);
        }
    }
    // join the row groups of the wave, then the waves
    auto add = [](float x, float y) { return x + y; };
    auto larger = [](float x, float y) { return fmaxf(x, y); };
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const float mn = over_rows<LPR>(m[g], larger);
        const float ref = mn == -INFINITY ? 0.f : mn, f = __builtin_amdgcn_exp2f(m[g] - ref);
        const float ls = over_rows<LPR>(l[g] * f, add);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float t = over_rows<LPR>(o[g][e] * f, add);
            if (lane < LPR) so[wave][g][ch * E + e] = t;
        }
        if (lane == 0) {
            sm[wave][g] = mn;
            sl[wave][g] = ls;
        }
    }
    __syncthreads();
    for (int i = tid; i < ng * HD; i += NT) {
        const int g = i / HD, d = i % HD;
        float mn = sm[0][g];
#pragma unroll
        for (int w = 1; w < NW; ++w) mn = fmaxf(mn, sm[w][g]);
        const float ref = mn == -INFINITY ? 0.f : mn;
        float ls = 0.f, t = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = __builtin_amdgcn_exp2f(sm[w][g] - ref);
            ls += sl[w][g] * f;
            t += so[w][g][d] * f;
        }
        if (a.splits == 1) {
            Act<T>::st((T*)a.out + ((int64_t)b * a.H + h0 + g) * HD + d, seen.vis > 0 ? t / ls : 0.f);
        } else {
            float* w = a.ws + (((int64_t)b * a.H + h0 + g) * a.splits + split) * (HD + 2);
            w[d] = t;
            if (d == 0) {       // an idle entry: weights of one, so that the join divides its zeros by something
                w[HD] = seen.vis > 0 ? mn : 0.f;
                w[HD + 1] = seen.vis > 0 ? ls : 1.f;
            }
        }
    }
}

// The splits (at most 64) of one (sequence, query head): a block per row.  Groups of HD / 2 threads take every GR-th split, all on their way before
// the weights are known; the groups are added in their order.  (32 rows of 128 from 64 splits: 3.8 us; a wave per row that walks the splits eight at
// a time 14 us.)
template <typename T, int HD>
__global__ __launch_bounds__(KT_) void step_join_kernel(const float* __restrict__ ws, T* __restrict__ out, int splits) {
    constexpr int TR = HD / 2, GR = KT_ / TR, K = 64 / GR > 0 ? 64 / GR : 1;
    __shared__ float sf[64];
    __shared__ float so[GR][HD];
    const int tid = threadIdx.x, lane = tid & 63, g = tid / TR, d = tid % TR * 2;
    const float* w = ws + (int64_t)blockIdx.x * splits * (HD + 2);
    float2 v[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int sp = k * GR + g;
        v[k] = sp < splits ? *reinterpret_cast<const float2*>(w + sp * (HD + 2) + d) : make_float2(0.f, 0.f);
    }
    if (tid < 64) {
        const float m = lane < splits ? w[lane * (HD + 2) + HD] : -INFINITY, l = lane < splits ? w[lane * (HD + 2) + HD + 1] : 0.f;
        const float mn = wave_max(m);
        const float f = __builtin_amdgcn_exp2f(m - mn);         // every score -inf: NaN, as without splits
        sf[lane] = f / wave_sum(l * f);
    }
    __syncthreads();
    float2 t = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int sp = k * GR + g;
        if (sp < splits) {
            t.x = __builtin_fmaf(sf[sp], v[k].x, t.x);
            t.y = __builtin_fmaf(sf[sp], v[k].y, t.y);
        }
    }
    so[g][d] = t.x;
    so[g][d + 1] = t.y;
    __syncthreads();
    if (tid < HD) {
        float r = 0.f;
#pragma unroll
        for (int i = 0; i < GR; ++i) r += so[i][tid];
        Act<T>::st(out + (int64_t)blockIdx.x * HD + tid, r);
    }
}

// ------------------------------------------------------------------------------------------------------
extern "C" int star_kv_append(const void* qkv, int64_t ld, const int64_t* offsets, void* cache, const int32_t* lengths, int64_t R, int NB, int L,
                              int H, int KV, int hd, int cap, int sinks, int dt, void* stream) {
    STAR_CHECK(qkv && cache && lengths, "star_kv_append: null pointer");
    STAR_CHECK(dt == STAR_BF16 || dt == STAR_F32, "star_kv_append: dtype %d is neither STAR_BF16 nor STAR_F32", dt);
    const int es = dt == STAR_BF16 ? 2 : 4;
    STAR_CHECK(NB > 0 && NB <= 65535 && L >= 0 && H > 0 && KV > 0 && hd > 0 && hd % 8 == 0 && (int64_t)(H + 2 * (int64_t)KV) * hd <= ld && hd <= 65536 && KV <= 65536,
               "star_kv_append: bad shape NB=%d L=%d H=%d KV=%d hd=%d ld=%lld", NB, L, H, KV, hd, (long long)ld);
    STAR_CHECK(cap <= (1 << 30) && L <= (1 << 30), "star_kv_append: a cache of %d slots, sequences of %d", cap, L);
    STAR_CHECK(sinks >= 0 && cap > sinks, "star_kv_append: a cache of %d slots does not hold %d sinks and a ring", cap, sinks);
    STAR_CHECK(R >= 0 && (offsets || R == (int64_t)NB * L), "star_kv_append: %lld rows for %d sequences of %d", (long long)R, NB, L);
    STAR_CHECK(ld * es % 16 == 0 && (uintptr_t)qkv % 16 == 0 && (uintptr_t)cache % 16 == 0, "star_kv_append: rows and cache must be 16-byte aligned");
    STAR_CHECK(!star_meets(cache, 2 * (int64_t)NB * KV * cap * hd * es, qkv, R, ld * es, ((int64_t)H + 2 * (int64_t)KV) * hd * es), "star_kv_append: cache overlaps qkv");
    if (L == 0 || R == 0) return 0;
    if (L > R) L = (int)R;          // ragged: no sequence has more
    const AppendArgs a = {qkv, offsets, cache, lengths, ld, R, NB, L, H, KV, hd, cap, sinks};
    const int64_t chunks = (int64_t)L * 2 * KV * (hd * es / 16);
    // Blocks of a sequence, for the longest of them.  Ragged with many sequences: fewer, since those of short ones end at once but are launched all the
    // same (one prompt of 200000 rows, 2 heads of 64, among 4095 idle entries: 4096 blocks each 4.96 ms, so 0.14; 200 prompts of 700 rows, 8 heads: 103.0
    // and 103.0 us, 2000 of 100: 150.7 and 150.6).
    const int64_t want = (chunks + KT_ - 1) / KT_, share = !offsets || NB < 32 ? 4096 : 131072 / NB < 16 ? 16 : 131072 / NB;
    const dim3 grid((unsigned)(want < share ? want : share), NB);
    hipStream_t s = (hipStream_t)stream;
    if (dt == STAR_BF16) hipLaunchKernelGGL(kv_append_kernel<2>, grid, dim3(KT_), 0, s, a);
    else hipLaunchKernelGGL(kv_append_kernel<4>, grid, dim3(KT_), 0, s, a);
    STAR_LAUNCH_CHECK("star_kv_append");
    return 0;
}

// Query heads of a key head that one block serves: they share every row it reads, but its one or two rounds of rows cost the more arithmetic.  More
// than two only where the key heads alone fill the chip (1 sequence, 32 heads of 128 on 8, 1000 tokens: 11.8 us with four, 9.1 with two, 8.5 with one; 16 x
// 8 heads of 64 on 1, 2000 tokens: 12.8, 11.7, 11.0; 8 x 32 on 8, 4096 tokens: 33.6, 31.5, 82.3).  Eight for groups over four heads, or four where the
// sequences are split and four twice hold the group (64 x 64 heads of 128 on 8, 4096 tokens: 318 us with eight, 340 with four, 407 with two; 64 x 64 of 64 on
// 8, 500 tokens: 36, 47; 260 x 32 of 64 on 2, 1500 tokens, split: 129, 163; but 34 x 64 of 64 on 8, 2400 tokens, split: 73, 59, 63; 300 x 8 of 128 on 1,
// 1000 tokens, split: 78, 59).
static int step_group(int NB, int H, int KV) {
    const int rep = H / KV;
    if ((int64_t)NB * KV < star_num_cus()) return rep > 1 ? 2 : 1;
    return rep > 4 ? 8 : rep > 2 ? 4 : rep;
}
// Threads of a block and splits.  A wide block takes a whole sequence, in one launch, where three rounds of its rows hold it (5 sequences, 12 heads of
// 64, 1000 tokens: 8.6 us against 8.1 with narrow blocks, splits and their join, but a second launch takes the host 4 us longer: 10.4 against 14.6
// called one by one), and where the blocks fill every round of the compute units to nine tenths (64 sequences, 12 heads of 64, 1000 tokens: equal).
// Else narrow blocks, the tokens split until there are about four per compute unit for few (sequence, key head) pairs, eight for many (8 sequences,
// 32 heads on 8 of 128, 1000 tokens 14.9 us against 18.2 with eight; 33 x 8 heads of 128, 6000 tokens 152 us, 195 with whole sequences, which
// leave the second round of compute units nearly empty); no more splits than hold rows.
struct StepPlan {
    int group, threads, splits;
};
static StepPlan step_plan(int NB, int H, int KV, int hd, int es, int cap, int left, int sinks) {
    const int rep = H / KV;
    int G = step_group(NB, H, KV);
    const int wide = G == 8 ? 512 : 1024;
    int64_t blocks = (int64_t)NB * KV * cdiv(rep, G);
    const int64_t vis = (int64_t)left + 1 + sinks < cap ? (int64_t)left + 1 + sinks : cap;
    const int per = 4 * 64 / (hd * es / 16);              // rows of a wave's round
    const int64_t cus = star_num_cus();
    if (vis <= 3 * per * (wide / 64) || (blocks >= cus && blocks * 10 >= cdiv(blocks, cus) * cus * 9)) return {G, wide, 1};
    if (G == 8 && rep <= 8) {
        G = 4;
        blocks *= 2;
    }
    const int64_t rounds = (vis + per * 4 - 1) / (per * 4);
    int64_t s = ((blocks < cus ? 4 : 8) * cus + blocks - 1) / blocks;
    s = s < 1 ? 1 : s > 64 ? 64 : s > rounds ? rounds : s;
    const int64_t each = (rounds + s - 1) / s;
    return {G, KT_, (int)((rounds + each - 1) / each)};
}

extern "C" int64_t star_attn_window_step_ws(int NB, int H, int KV, int hd, int cap, int left, int sinks, int dt) {
    if (NB <= 0 || H <= 0 || KV <= 0 || H % KV || hd < 16 || hd > 128 || cap <= 0 || left < 0 || sinks < 0) return 0;
    const int s = step_plan(NB, H, KV, hd, dt == STAR_BF16 ? 2 : 4, cap, left, sinks).splits;
    return s == 1 ? 0 : (int64_t)NB * H * s * (hd + 2);
}

template <typename T, int HD, int G> static void step_launch(const StepArgs& a, int threads, dim3 grid, hipStream_t s) {
    constexpr int WIDE = G == 8 ? 512 : 1024;
    if (threads == WIDE) hipLaunchKernelGGL((step_kernel<T, HD, G, WIDE>), grid, dim3(WIDE), 0, s, a);
    else hipLaunchKernelGGL((step_kernel<T, HD, G, KT_>), grid, dim3(KT_), 0, s, a);
}
template <typename T, int HD> static void step_heads(const StepArgs& a, int G, int threads, dim3 grid, hipStream_t s) {
    if (G == 1) step_launch<T, HD, 1>(a, threads, grid, s);
    else if (G == 2) step_launch<T, HD, 2>(a, threads, grid, s);
    else if (G == 4) step_launch<T, HD, 4>(a, threads, grid, s);
    else step_launch<T, HD, 8>(a, threads, grid, s);
    if (a.splits > 1) hipLaunchKernelGGL((step_join_kernel<T, HD>), dim3((unsigned)(a.NB * a.H)), dim3(KT_), 0, s, a.ws, (T*)a.out, a.splits);
}
template <typename T> static void step_run(const StepArgs& a, int hd, int G, int threads, dim3 grid, hipStream_t s) {
    if (hd == 16) step_heads<T, 16>(a, G, threads, grid, s);
    else if (hd == 32) step_heads<T, 32>(a, G, threads, grid, s);
    else if (hd == 64) step_heads<T, 64>(a, G, threads, grid, s);
    else step_heads<T, 128>(a, G, threads, grid, s);
}

extern "C" int star_attn_window_step(const StarAttnStep* g, void* stream) {
    STAR_CHECK(g && g->qkv && g->cache && g->lengths && g->out, "star_attn_window_step: null pointer");
    STAR_CHECK(g->dt == STAR_BF16 || g->dt == STAR_F32, "star_attn_window_step: dtype %d is neither STAR_BF16 nor STAR_F32", g->dt);
    const int es = g->dt == STAR_BF16 ? 2 : 4;
    STAR_CHECK(g->hd == 16 || g->hd == 32 || g->hd == 64 || g->hd == 128, "star_attn_window_step: head dim %d not in {16,32,64,128}", g->hd);
    STAR_CHECK(g->NB > 0 && g->H > 0 && g->KV > 0 && g->H % g->KV == 0 && g->H <= 65536 / g->hd, "star_attn_window_step: bad shape NB=%d H=%d KV=%d", g->NB, g->H, g->KV);
    STAR_CHECK(g->sinks >= 0 && g->left >= 0 && (int64_t)g->sinks + g->left < g->cap, "star_attn_window_step: a cache of %d slots does not hold %d sinks and a window of %d + 1",
               g->cap, g->sinks, g->left);
    STAR_CHECK(g->cap <= (1 << 30), "star_attn_window_step: a cache of %d slots", g->cap);
    STAR_CHECK(g->scale > 0.f && g->scale < INFINITY, "star_attn_window_step: scale %g must be positive", (double)g->scale);
    STAR_CHECK(g->ld >= (int64_t)(g->H + 2 * g->KV) * g->hd && g->ld * es % 16 == 0 && (uintptr_t)g->qkv % 16 == 0 && (uintptr_t)g->cache % 16 == 0,
               "star_attn_window_step: rows must hold all heads, rows and cache must be 16-byte aligned");
    StepArgs a = {g->qkv, g->cache, g->lengths, g->pos, g->out, g->ws, g->ld, g->pos_ld, g->NB, g->H, g->KV, g->cap, g->left, g->sinks, 1, 1, g->scale * LOG2E, {}};
    if (g->h_rope) {
        const int n = g->h_rope->pairs;
        STAR_CHECK(g->pos && g->pos_ld >= g->NB, "star_attn_window_step: a rotation needs positions of every sequence");
        STAR_CHECK(n > 0 && n <= 64 && 2 * n <= g->hd && g->h_rope->axes > 0, "star_attn_window_step: %d pairs in heads of %d", n, g->hd);
        for (int i = 0; i < n; ++i)
            STAR_CHECK(g->h_rope->axis[i] < g->h_rope->axes, "star_attn_window_step: pair %d turns by axis %d of %d", i, g->h_rope->axis[i], g->h_rope->axes);
        a.f = *g->h_rope;
    }
    const StepPlan plan = step_plan(g->NB, g->H, g->KV, g->hd, es, g->cap, g->left, g->sinks);
    const int G = plan.group;
    a.chunks = cdiv(g->H / g->KV, G);
    a.splits = plan.splits;
    STAR_CHECK(a.splits == 1 || g->ws, "star_attn_window_step: null workspace (star_attn_window_step_ws)");
    const int64_t blocks = ((int64_t)g->NB * g->KV * a.splits + 7) / 8 * 8 * a.chunks;
    // the hardware counts a launch's threads in 32 bits
    STAR_CHECK(blocks * plan.threads < (1ll << 32) && (a.splits == 1 || (int64_t)g->NB * g->H * KT_ < (1ll << 32)), "star_attn_window_step: NB, H too large for the grid");
    // (a single row in place: the blocks of a head alone read its query)
    const int64_t out_bytes = (int64_t)g->NB * g->H * g->hd * es, cache_bytes = 2 * (int64_t)g->NB * g->KV * g->cap * g->hd * es, row = (int64_t)(g->H + 2 * g->KV) * g->hd * es;
    const int64_t ws_bytes = a.splits == 1 ? 0 : (int64_t)g->NB * g->H * a.splits * (g->hd + 2) * 4;
    auto meets = [&](const void* p, int64_t n) { return star_meets(p, n, g->qkv, g->NB, g->ld * es, row); };
    STAR_CHECK((g->NB == 1 && g->out == g->qkv) || !meets(g->out, out_bytes), "star_attn_window_step: out overlaps qkv");
    STAR_CHECK(!meets(g->cache, cache_bytes) && !star_meets(g->cache, cache_bytes, g->out, out_bytes), "star_attn_window_step: cache overlaps qkv or out");
    STAR_CHECK(!meets(g->ws, ws_bytes) && !star_meets(g->ws, ws_bytes, g->out, out_bytes) && !star_meets(g->ws, ws_bytes, g->cache, cache_bytes),
               "star_attn_window_step: ws overlaps another operand");
    hipStream_t s = (hipStream_t)stream;
    if (g->dt == STAR_BF16) step_run<bf16_t>(a, g->hd, G, plan.threads, dim3((unsigned)blocks), s);
    else step_run<float>(a, g->hd, G, plan.threads, dim3((unsigned)blocks), s);
    STAR_LAUNCH_CHECK("star_attn_window_step");
    return 0;
}
