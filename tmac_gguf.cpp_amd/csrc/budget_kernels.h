// budget_kernels.h -- kernels that keep long contexts in a small cache (part of
// paged_kernels.hip): 4-bit pages, append at given rows with rotary positions of
// several axes, attention that leaves the weight of every row, the rows to keep
// by it, and the compaction of a cache to those rows.

// ---------------------------------------------------------------------------
// 4-bit rows.  A block of 32 dims: the scale is the value of the largest
// magnitude over -8 (the negative one where both signs have it), so that it
// takes the code 0, rounded to 7 bits; a code is the nearest, ties to even.
// Magnitudes whose scale is below 2^-14 are 0; a scale above 8,128 is infinity,
// and a NaN makes the block's scale NaN.
__device__ __forceinline__ unsigned quant_codes(const float* x, float hi, float lo, bool bad, unsigned& dbits) {
    const float t = (hi > -lo ? hi : lo) * -0.125f;
    const unsigned u = __float_as_uint(t);
    float d = __uint_as_float((u + 0xFFFFu + ((u >> 17) & 1u)) & ~0x1FFFFu);
    d = fabsf(d) < 0x1p-14f ? 0.f : fabsf(d) > 8128.f ? d * -kNegInf : d;
    if (bad) d = __builtin_nanf("");
    dbits = __builtin_bit_cast(unsigned short, (_Float16)d);
    unsigned packed = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float q = fminf(fmaxf(__builtin_rintf(x[e] / d) + 8.f, 0.f), 15.f);
        packed |= (d == 0.f ? 8u : (unsigned)q) << (8 * e);
    }
    return packed;
}

// Rounds this lane's 8 dims (load8's) of row r and writes them to the (page, kv
// head) block at p.  The 8 lanes of a slot must all call.
__device__ __forceinline__ void put_row4(const float (&x)[8], char* p, int r, int c, bool key) {
    float hi[2], lo[2];
    int bad = 0;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const float* y = x + 4 * b;
        hi[b] = slot_max(fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])));
        lo[b] = -slot_max(-fminf(fminf(y[0], y[1]), fminf(y[2], y[3])));
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= (y[e] != y[e] ? 1 : 0) << b;
    }
    bad |= __shfl_xor(bad, 1);
    bad |= __shfl_xor(bad, 2);
    bad |= __shfl_xor(bad, 4);
    unsigned d[2], w[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) w[b] = quant_codes(x + 4 * b, hi[b], lo[b], bad >> b & 1, d[b]);
    unsigned char* q = reinterpret_cast<unsigned char*>(p);
    uint16_t* s = reinterpret_cast<uint16_t*>(p) + 256;
    if (key) {
        // dims 32 b + 4 c + e: bytes of the pairs (e, e + 2)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int g = 2 * b + (c >> 2), m = (c >> 1) & 1;
            unsigned char* o = q + 8 * (16 * g + r) + 4 * m + (c & 1);
            o[0] = (unsigned char)((w[b] & 15u) | (w[b] >> 16 & 15u) << 4);
            o[2] = (unsigned char)((w[b] >> 8 & 15u) | (w[b] >> 24 & 15u) << 4);
            if (c == 0) s[16 * b + r] = (uint16_t)d[b];
        }
    } else {
        // dims 4 c + e of half b, c < 4, pair with those of lane c + 4: lanes c < 4 write half 0, the others half 1
        const unsigned other = (unsigned)__shfl_xor((int)(c < 4 ? w[1] : w[0]), 4);
        const unsigned low = c < 4 ? w[0] : other, high = c < 4 ? other : w[1];
        const int pos = (r & 3) == 1 ? 2 : (r & 3) == 2 ? 1 : r & 3;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            q[8 * (16 * (r >> 2) + 4 * (c & 3) + e) + (c < 4 ? 0 : 4) + pos] =
                (unsigned char)((low >> (8 * e) & 15u) | (high >> (8 * e) & 15u) << 4);
        if ((c & 3) == 0) s[8 * (r >> 2) + 4 * (c >> 2) + (r & 3)] = (uint16_t)d[c >> 2];
    }
}

// This lane's 8 dims (load8's) of row r of the (page, kv head) block at p.
__device__ __forceinline__ void load_row4(float (&x)[8], const char* p, int r, int c, bool key) {
    const unsigned char* q = reinterpret_cast<const unsigned char*>(p);
    const uint16_t* s = reinterpret_cast<const uint16_t*>(p) + 256;
    const int pos = (r & 3) == 1 ? 2 : (r & 3) == 2 ? 1 : r & 3;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const float d = half_bits_to_float(key ? s[16 * b + r] : s[8 * (r >> 2) + 4 * b + (r & 3)]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int dim = 32 * b + 4 * c + e;
            int byte, high;
            if (key) {
                const int y = dim & 7;
                byte = 8 * (16 * (dim >> 4) + r) + 4 * (dim >> 3 & 1) + (y >> 2) + 2 * (y & 1);
                high = y >> 1 & 1;
            } else {
                byte = 8 * (16 * (r >> 2) + (dim & 15)) + 4 * b + pos;
                high = dim >> 4 & 1;
            }
            x[4 * b + e] = (float)((int)(q[byte] >> (4 * high) & 15) - 8) * d;
        }
    }
}

// ---------------------------------------------------------------------------
// Pages widened to fp32.  A workgroup takes a page's head, a slot of 8 lanes a
// row of K (first half of the slots) or V; 4-bit blocks come through LDS.  Bound by
// the fp32 rows it writes: 2 x 996 pages of 2 heads, 18 MB, 5.7 us of which 2 are
// the launch; 2 x 24,750 pages, 460 MB, 94 us = 4.9 TB/s, a large copy's rate.
template <typename T>
__device__ __forceinline__ void widen_body(const WidenArgs& a) {
    const int c = threadIdx.x & 7, r = threadIdx.x >> 3 & 15, v = threadIdx.x >> 7;
    const int64_t unit = blockIdx.x;
    const int page = (int)(unit / a.n_kv_head), h = (int)(unit - (int64_t)page * a.n_kv_head);
    const size_t at = (size_t)page * PageFmt<T>::page(a.n_kv_head) + PageFmt<T>::head(h);
    float x[8];
    if constexpr (__is_same(T, q4_t)) {
        __shared__ u32x4 s_block[2][kQ4Block / 16];  // (bytes one by one from memory: 7.3 us instead of 5.7)
        const int i = threadIdx.x & 127;
        if (a.pages[v] && i < kQ4Block / 16) s_block[v][i] = *reinterpret_cast<const u32x4*>(a.pages[v] + at + 16 * i);
        __syncthreads();
        if (!a.pages[v]) return;
        load_row4(x, reinterpret_cast<const char*>(s_block[v]), r, c, v == 0);
    } else {
        if (!a.pages[v]) return;
        load_row<T, false>(x, a.pages[v] + at + r * PageFmt<T>::row(a.n_kv_head) + 4 * c * CacheFmt<T>::kDimBytes, c);
    }
    store8(a.out[v] + (((size_t)page * kPageRows + r) * a.n_kv_head + h) * kHeadDim + 4 * c, x);
}

// ---------------------------------------------------------------------------
// Append at given rows.  The rows' sequences are found as in append_body; a
// pair (d, d + 1) turns by the position on its axis, so a lane reads the four
// (cos, sin) of its pairs from up to four table rows.  A 4-bit row is rounded by the
// 8 lanes that hold it.  Bound by memory: 15,829 rows of 14 + 2 + 2 heads into 4-bit
// pages, 136 MB, 25 us where they come again from the last-level cache (5.4 TB/s),
// 34.6 from memory (3.9; a large copy takes 27.8).  A wave has head rows of one kind:
// with q, k and v mixed every wave went through the rounding, 38.8.  Loads one or two
// head rows ahead, and (cos, sin) through LDS, took as long.  A single row is all
// latency, 3.2 us.
template <typename T>
__device__ __forceinline__ void append_axes_body(const AppendAxesArgs& x_args) {
    const AppendArgs& a = x_args.a;
    __shared__ int s_seq[kAppendRows];
    __shared__ int64_t s_page[kAppendRows];  // pool page, -1: not stored
    __shared__ int s_at[kAppendRows];        // row in the page, -1: the row is skipped
    __shared__ int s_pos[4][kAppendRows];    // position on each axis
    const int R = a.rows_per_group;
    const int t0 = blockIdx.x * R, n = min(R, a.n_rows - t0);
    const int tid = threadIdx.x;
    if (tid < kAppendRows) s_seq[tid] = -1;
    __syncthreads();
    for (int i = tid; i <= a.n_seq; i += 256) {
        const int at = a.row_starts[i];
        if (at <= t0)
            atomicMax(&s_seq[0], i);
        else if (at < t0 + n)
            atomicMax(&s_seq[at - t0], i);
    }
    __syncthreads();
    if (tid < n) {
        int s = -1;
        for (int i = 0; i <= tid; ++i) s = max(s, s_seq[i]);
        int at = -1;
        int64_t page = -1;
        if (s >= 0 && s < a.n_seq) {  // entry n_seq: rows behind the last sequence
            bool ok = true;
            for (int i = 0; i < x_args.n_axes; ++i) {
                const int p = x_args.pos[(size_t)i * a.n_rows + t0 + tid];
                ok &= (unsigned)p < (unsigned)x_args.max_pos;
                s_pos[i][tid] = p;
            }
            const int64_t row = (int64_t)a.positions[s] + (t0 + tid - a.row_starts[s]);
            if (ok && row >= 0 && row < a.capacity) {
                at = (int)row & (kPageRows - 1);
                page = a.block_table[(size_t)s * a.max_pages + (row >> kPageShift)];
                if (page < 0 || page >= a.n_pages) {
                    page = -1;
                    atomicOr(a.err, 4);
                }
            } else {
                atomicOr(a.err, 1);
            }
        }
        s_at[tid] = at;
        s_page[tid] = page;
    }
    __syncthreads();
    const int c = tid & 7, slot = tid >> 3;
    // Head rows of q, then of k, then of v, each from a wave's first slot on: a wave has one kind.
    const int nh = a.q ? a.n_head : 0, kv = a.n_kv_head, nq = n * nh, nk = n * kv, q8 = (nq + 7) & ~7, k8 = (nk + 7) & ~7;
    for (int it = slot; it < q8 + 2 * k8; it += 32) {
        const bool query = it < q8, key = it < q8 + k8;
        const int i = query ? it : key ? it - q8 : it - q8 - k8, heads = query ? nh : kv;
        if (i >= (query ? nq : nk)) continue;
        const int r = i / heads, h = i - r * heads, at = s_at[r];
        if (at < 0) continue;
        const int64_t t = t0 + r, page = s_page[r];
        float x[8];
        auto turn = [&]() {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int pair = (i < 2 ? 0 : 16) + 2 * c + (i & 1);
                const int axis = (int)(x_args.pair_axis >> (2 * pair)) & 3;
                const float2 cs = a.rope_cs[(size_t)s_pos[axis][r] * (kHeadDim / 2) + pair];
                rotate_pair(x[2 * i], x[2 * i + 1], cs.x, cs.y);
            }
        };
        if (query) {
            load8(x, a.q + t * a.q_stride + (int64_t)h * kHeadDim + 4 * c);
            turn();
            store8(a.q_out + (t * nh + h) * kHeadDim + 4 * c, x);
        } else if (page >= 0) {
            load8(x, (key ? a.k + t * a.k_stride : a.v + t * a.v_stride) + (int64_t)h * kHeadDim + 4 * c);
            if (key) turn();
            char* p = (key ? a.k_pages : a.v_pages) + (size_t)page * PageFmt<T>::page(kv) + PageFmt<T>::head(h);
            if constexpr (__is_same(T, q4_t))
                put_row4(x, p, at, c, key);
            else
                put_row<T>(x, p + at * PageFmt<T>::row(kv) + 4 * c * CacheFmt<T>::kDimBytes, c, true);
        }
    }
}

// ---------------------------------------------------------------------------
// Attention over 4-bit pages: two pages a step, 32 keys, on the fp16 products of
// fp16 rows (two parts of q and of the weights).  Both operands come from memory
// in their lanes.  A word of 8 codes: a mask and an or make each pair of codes
// n the fp16 pair 1024 + n (codes in the high half of a byte: 1024 + 16 n), a
// subtraction (a fma: a sixteenth, minus 72) n - 8, and a product with the scale
// the pair of values, all exact.
// A step of 7 heads is 188 vector instructions and 8 products, which do not overlap:
// some 930 cycles of a SIMD.  256 sequences of up to 4,096 rows (14 heads on 2,
// 117 MB) take 29.4 us, 4.0 TB/s where a large copy reaches 4.9; instructions fill
// two thirds of that time.
struct Codes {
    using M = MMath<_Float16>;
    struct Tile {
        u32x2 k, v;
        unsigned kd;  // scales of rows lane % 16 & ~1, | 1, dims 16 (lane / 16) .. (16 bits alone are widened where
                      // the loop waits for them)
        u32x4 vd;     // scales of rows 4 (lane / 16) .. of dims 0 .. 31, then 32 .. 63
    };
    __device__ static void fetch(Tile& t, const char* kp, const char* vp, int lane) {
        // Through descriptors of one block each: offsets of 32 bits beside a scalar base.
        auto block = [](const char* p) {
            return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p), 0, kQ4Block, 0x00020000);
        };
        const auto kb = block(kp), vb = block(vp);
        t.k = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(kb, 8 * lane, 0, 0));
        t.v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(vb, 8 * lane, 0, 0));
        t.kd = __builtin_amdgcn_raw_buffer_load_b32(kb, 32 * (lane >> 5) + 4 * ((lane & 15) >> 1), 512, 0);
        t.vd = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(vb, 16 * (lane >> 4), 512, 0));
    }
    // Weights come up to 2^15, so that their low parts stay in fp16's normal range without a product of their own.
    static constexpr int kGain = 7;
    // Masks in scalar registers and the ones in a vector register make mask and or one instruction (as plain constants
    // two, 32 more a step); minus one makes x - (float)half one mixed fma (as a constant a conversion and a difference).
    unsigned low_mask = 0x000F000Fu, high_mask = 0x00F000F0u, one = 0x64006400u;
    float minus = -1.f;
    __device__ Codes() { asm("" : "+s"(low_mask), "+s"(high_mask), "+v"(one), "+s"(minus)); }
    __device__ f16x2 low(unsigned w) const {
        const f16x2 bias = {(_Float16)1032.0f, (_Float16)1032.0f};
        return __builtin_bit_cast(f16x2, (w & low_mask) | one) - bias;
    }
    __device__ f16x2 high(unsigned w) const {
        const f16x2 sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f}, bias = {(_Float16)-72.0f, (_Float16)-72.0f};
        return __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (w & high_mask) | one), sixteenth, bias);
    }
    // The K operand of depth block m: dims 16 g + 8 m + 0..7 of row lane % 16.
    __device__ f16x2 key_scale(const Tile& t, int lane) const {
        const _Float16 d = __builtin_bit_cast(_Float16, (unsigned short)(t.kd >> (16 * (lane & 1))));
        return f16x2{d, d};
    }
    __device__ M::v8 key(const Tile& t, int m, f16x2 d0) const {
        const unsigned x = t.k[m], y = x >> 8;
        const f16x2 e[4] = {low(x) * d0, high(x) * d0, low(y) * d0, high(y) * d0};
        return __builtin_bit_cast(M::v8, e);
    }
    // The V operands of dims 32 p + i, 32 p + 16 + i: rows 4 g + 0..3 of both pages.
    __device__ void values(M::v8 (&x)[2], const Tile (&t)[2], int p) const {
        f16x2 e[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const unsigned w = t[u].v[p], y = w >> 8;
            // (a copy first: the bit cast of a vector's element reads the vector's first one)
            const unsigned a0 = t[u].vd[2 * p], b0 = t[u].vd[2 * p + 1];
            const f16x2 a = __builtin_bit_cast(f16x2, a0), b = __builtin_bit_cast(f16x2, b0);
            e[0][2 * u] = low(w) * a;
            e[0][2 * u + 1] = low(y) * b;
            e[1][2 * u] = high(w) * a;
            e[1][2 * u + 1] = high(y) * b;
        }
        x[0] = __builtin_bit_cast(M::v8, e[0]);
        x[1] = __builtin_bit_cast(M::v8, e[1]);
    }
    // Two weights as their two parts.
    __device__ void parts(float x, float y, unsigned& top, unsigned& rest) const {
        top = M::pack2(x, y);
        asm("" : "+v"(top));  // (one conversion of the pair, not one more of each)
        const f16x2 t = __builtin_bit_cast(f16x2, top);
        rest = M::pack2(__builtin_fmaf((float)t[0], minus, x), __builtin_fmaf((float)t[1], minus, y));
    }
    // Scales of V with those of the rows outside lo .. hi - 1 as zeros (a row outside may hold any).
    __device__ static u32x4 rows_in(u32x4 vd, int lo, int hi, int g) {
        auto in = [&](int r) { return 4 * g + r >= lo && 4 * g + r < hi; };
        const unsigned m0 = (in(0) ? 0xFFFFu : 0u) | (in(1) ? 0xFFFF0000u : 0u);
        const unsigned m1 = (in(2) ? 0xFFFFu : 0u) | (in(3) ? 0xFFFF0000u : 0u);
        return u32x4{vd[0] & m0, vd[1] & m1, vd[2] & m0, vd[3] & m1};
    }
    // Dims 16 g + 8 m + 0..7 of a query.
    __device__ static void query(RawQ<_Float16, Mfma16>& q, const float* p, int lane) {
        const int g = lane >> 4;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                q.x[m][i] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (p) q.x[m][i] = *reinterpret_cast<const f32x4*>(p + 16 * g + 8 * m + 4 * i);
            }
    }
};

// Up to 16 query heads a kv head: a column each, the parts as products of their own, 16 a step.
template <>
struct Own<q4_t> {
    using S = Mfma16;
    using State = Cols<_Float16, S>;
    using RawQuery = RawQ<_Float16, S>;
    using Tile = Codes::Tile;
    static constexpr int kTiles = 2;
    struct Lds {};
    __device__ static int column(int lane) { return lane & 15; }
    __device__ static void query(RawQuery& q, const float* p, int lane) { Codes::query(q, p, lane); }
    __device__ static void init(State& st, const RawQuery& q, float scale) { cols_init<_Float16, S>(st, q, scale); }
    __device__ static void fetch(Tile& t, const char* kp, const char* vp, size_t, int lane) { Codes::fetch(t, kp, vp, lane); }
    // Keys lo[u] .. hi[u] - 1 of page u take part.
    template <typename Score>
    __device__ static void attend(State& st, Tile (&t)[kTiles], const int (&lo)[kTiles], const int (&hi)[kTiles], Lds&,
                                  int lane, Score score) {
        using M = MMath<_Float16>;
        const Codes k;
        const int g = lane >> 4;
        f32x4 w[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const f16x2 d = k.key_scale(t[u], lane);
            w[u] = score_tile<_Float16, S>(st, nullptr, nullptr, g, [&](int m, int) { return k.key(t[u], m, d); });
        }
        if (!(lo[0] <= 0 && lo[1] <= 0 && hi[0] >= kPageRows && hi[1] >= kPageRows)) {
            asm volatile("");  // a branch, not selects
#pragma unroll
            for (int u = 0; u < 2; ++u) {
#pragma unroll
                for (int r = 0; r < 4; ++r) w[u][r] = 4 * g + r >= lo[u] && 4 * g + r < hi[u] ? w[u][r] : kNegInf;
                t[u].vd = Codes::rows_in(t[u].vd, lo[u], hi[u], g);
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) score(u, w[u] + st.base);
        softmax_step<S, Codes::kGain>(st.m, st.l, st.base, st.o, w);
        u32x4 p[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                unsigned top, rest;
                k.parts(w[u][2 * r], w[u][2 * r + 1], top, rest);
                p[0][2 * u + r] = top;
                p[1][2 * u + r] = rest;
            }
        const M::v8 px[2] = {__builtin_bit_cast(M::v8, p[0]), __builtin_bit_cast(M::v8, p[1])};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            M::v8 x[2];
            k.values(x, t, h);
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 2; ++i) st.o[2 * h + b] = M::mfma32(x[b], px[i], st.o[2 * h + b]);
        }
    }
    __device__ static void finish(State& st) { st.l *= 1.0f / (1 << Codes::kGain); }
    static constexpr int dim(int b, int g) { return 16 * b + 4 * g; }
    __device__ static f32x4 sums(const State& st, int b) { return st.o[b] * (1.0f / (1 << Codes::kGain)); }
};

// Up to 8 query heads a kv head: column c < 8 holds the first part of head c, column
// c + 8 the second, of q and of the weights, so that a product takes both (8 a step
// instead of 16, which cost the SIMD 16 cycles each beside the other instructions, not
// under them).  A score is the sum of two columns; lane c goes on with page 0 and
// lane c + 8 with page 1 of the step, half the exponentials each.  (256 sequences as
// above: 29.2 us instead of 33.8 by the form for 16 heads; one of 700 rows 6.1, both.)
template <>
struct Own<q4_pair_t> {
    using S = Mfma16;
    using M = MMath<_Float16>;
    using RawQuery = RawQ<_Float16, S>;
    using Tile = Codes::Tile;
    static constexpr int kTiles = 2;
    struct State {
        M::v8 q[2];
        f32x4 o[4];
        float unscale, m, l, base;
    };
    struct Lds {};
    __device__ static int column(int lane) { return lane & 7; }
    __device__ static float across(float x) { return dpp<0x128>(x); }  // of lane ^ 8
    __device__ static unsigned across(unsigned x) { return dpp_u<0x128>(x); }
    __device__ static void query(RawQuery& q, const float* p, int lane) { Codes::query(q, p, lane); }
    __device__ static void init(State& st, const RawQuery& q, float scale) {
        Cols<_Float16, S> c;
        cols_init<_Float16, S>(c, q, scale);
        const bool first = !(threadIdx.x & 8);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const u32x4 a = __builtin_bit_cast(u32x4, c.q[m][0]), b = __builtin_bit_cast(u32x4, c.q[m][1]);
            u32x4 x;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = first ? a[i] : b[i];
            st.q[m] = __builtin_bit_cast(M::v8, x);
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) st.o[b] = f32x4{0.f, 0.f, 0.f, 0.f};
        st.unscale = c.unscale;
        st.m = kNoMax;
        st.l = st.base = 0.f;
    }
    __device__ static void fetch(Tile& t, const char* kp, const char* vp, size_t, int lane) { Codes::fetch(t, kp, vp, lane); }
    template <typename Score>
    __device__ static void attend(State& st, Tile (&t)[kTiles], const int (&lo)[kTiles], const int (&hi)[kTiles], Lds&,
                                  int lane, Score score) {
        const Codes k;
        const int g = lane >> 4;
        const bool first = !(lane & 8);
        f32x4 acc[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const f16x2 d = k.key_scale(t[u], lane);
            acc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int m = 0; m < 2; ++m) acc[u] = M::mfma32(k.key(t[u], m, d), st.q[m], acc[u]);
        }
        f32x4 w;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float a = acc[0][r] + across(acc[0][r]), b = acc[1][r] + across(acc[1][r]);
            w[r] = __builtin_fmaf(first ? a : b, st.unscale, -st.base);
        }
        if (!(lo[0] <= 0 && lo[1] <= 0 && hi[0] >= kPageRows && hi[1] >= kPageRows)) {
            asm volatile("");  // a branch, not selects
            const int from = first ? lo[0] : lo[1], to = first ? hi[0] : hi[1];
#pragma unroll
            for (int r = 0; r < 4; ++r) w[r] = 4 * g + r >= from && 4 * g + r < to ? w[r] : kNegInf;
#pragma unroll
            for (int u = 0; u < 2; ++u) t[u].vd = Codes::rows_in(t[u].vd, lo[u], hi[u], g);
        }
        score(first ? 0 : 1, w + st.base);
        // as softmax_step, a column's maximum over its lanes of both pages
        const int over = max(max((int)__float_as_uint(w[0]), (int)__float_as_uint(w[1])),
                             max((int)__float_as_uint(w[2]), (int)__float_as_uint(w[3])));
        if (__any(over > (int)__float_as_uint(kTau + Codes::kGain) || st.m == kNoMax)) {
            float top = fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3]));
            top = max4_rows(top);
            top = fmaxf(top, across(top));
            const float m1 = fmaxf(st.m, st.base + top);
            const float b1 = m1 == kNoMax ? 0.f : m1 - Codes::kGain, shift = b1 - st.base;
            const float f = fast_exp2(st.m - m1);
            st.m = m1;
            st.base = b1;
            st.l *= f;
#pragma unroll
            for (int b = 0; b < 4; ++b) st.o[b] *= f;
            w -= shift;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r] = fast_exp2(w[r]);
        st.l += (w[0] + w[1]) + (w[2] + w[3]);
        unsigned p[4];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            unsigned top, rest;
            k.parts(w[2 * r], w[2 * r + 1], top, rest);
            const unsigned got = across(first ? rest : top);  // the other page's part that this column holds
            p[r] = first ? top : got;
            p[2 + r] = first ? got : rest;
        }
        const M::v8 px = __builtin_bit_cast(M::v8, u32x4{p[0], p[1], p[2], p[3]});
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            M::v8 x[2];
            k.values(x, t, h);
#pragma unroll
            for (int b = 0; b < 2; ++b) st.o[2 * h + b] = M::mfma32(x[b], px, st.o[2 * h + b]);
        }
    }
    // Both columns of a head get its sums.
    __device__ static void finish(State& st) {
        st.l = (st.l + across(st.l)) * (1.0f / (1 << Codes::kGain));
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) st.o[b][r] += across(st.o[b][r]);
    }
    static constexpr int dim(int b, int g) { return 16 * b + 4 * g; }
    __device__ static f32x4 sums(const State& st, int b) { return st.o[b] * (1.0f / (1 << Codes::kGain)); }
};

template <typename T>
constexpr bool kPages4 = __is_same(T, q4_t) || __is_same(T, q4_pair_t);
// The query head that this lane's column is of.
template <typename T>
__device__ __forceinline__ int column_of(int lane) {
    if constexpr (kPages4<T>)
        return Own<T>::column(lane);
    else
        return lane & 15;
}

// ---------------------------------------------------------------------------
// Attention over whole sequences, and the weights that rows get: w_r = sum over the
// heads of exp(s_r - M) / L, for which a row's scores wait until M and L are known.
// A workgroup of 8 waves takes a (sequence, kv head) whole, in one launch, or a share
// of it, and a second launch joins.  Read once, rows cost what memory gives: 256
// sequences of up to 4,096 rows, 14 heads on 2: bf16 81 us (5.0 TB/s), fp32 157 (5.2);
// Q8_0 and 4-bit rows the unpacking, 77 (2.9) and 29.4 (4.0).  One of 700 4-bit rows
// 6.0, a launch being 3.

// A sequence's length in rows, -1 where it is longer than the launch covers.
__device__ __forceinline__ int rows_of(const RowsArgs& a, int s) {
    const int len = max(a.lengths[s], 0);
    return len > a.max_len ? -1 : len;
}

enum class Scores { kNone, kFar, kNear };  // where they go: memory, LDS (near)

// Rows lo .. hi - 1 (lo at a step's start) of one (sequence, kv head): this wave's
// steps of kTiles pages, every BY-th from step `wave` on.  It looks up 64 pages at
// a time, and holds one step while the next is in flight (two in flight, or 16 waves,
// took as long).
template <typename T, int BY, Scores SCORES>
__device__ __forceinline__ void rows_attend(const RowsArgs& a, typename Own<T>::State& st, typename Own<T>::Lds& lds, int s,
                                            int h, int lo, int hi, int wave, int lane, float* near) {
    using O = Own<T>;
    constexpr int KT = O::kTiles;
    const int G = a.group, col = column_of<T>(lane);
    const int64_t row0 = (int64_t)s * a.n_head + h * G;
    typename O::RawQuery raw;
    O::query(raw, col < G ? a.q + (row0 + col) * kHeadDim : nullptr, lane);
    const size_t stride = PageFmt<T>::row(a.n_kv_head), page_bytes = PageFmt<T>::page(a.n_kv_head), head = PageFmt<T>::head(h);
    const int32_t* table = a.block_table + (size_t)s * a.max_pages + (lo >> kPageShift);
    float* const scores = a.scores + row0 * a.score_stride + (int64_t)lo * G;
    const int score_at = col < G ? 4 * (kPageRows * col + 4 * (lane >> 4)) : 1 << 30;  // (behind the range: dropped)
    const int rows = hi - lo, n = (rows + kPageRows - 1) >> kPageShift;
    const int steps = ((n + KT - 1) / KT - wave + BY - 1) / BY;  // this wave's
    for (int s0 = 0; s0 < steps; s0 += 64 / KT) {
        const int cnt = min(64 / KT, steps - s0);
        int page = 0;
        const int e = ((s0 + lane / KT) * BY + wave) * KT + lane % KT;
        if (lane < cnt * KT && e < n) {
            page = table[e];
            if (page < 0 || page >= a.n_pages) {
                atomicOr(a.err, 4);
                page = min(max(page, 0), a.n_pages - 1);
            }
        }
        typename O::Tile t[2][KT];
        auto fetch = [&](typename O::Tile (&x)[KT], int step) {
#pragma unroll
            for (int u = 0; u < KT; ++u) {
                const size_t at = (size_t)(unsigned)__builtin_amdgcn_readlane(page, KT * step + u) * page_bytes + head;
                O::fetch(x[u], a.k_pages + at, a.v_pages + at, stride, lane);
            }
        };
        fetch(t[0], 0);
        if (s0 == 0) O::init(st, raw, a.qscale);
        for (int step = 0; step < cnt; step += 2) {
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                if (step + d < cnt) {
                    // The last step is fetched again behind itself: under a condition, the wait for this step's rows would
                    // be one for all loads, the next step's among them.
                    fetch(t[1 - d], min(step + d + 1, cnt - 1));
                    const int r0 = ((s0 + step + d) * BY + wave) * KT * kPageRows, left = rows - r0;
                    int from[KT], to[KT];
#pragma unroll
                    for (int u = 0; u < KT; ++u) {
                        from[u] = 0;
                        to[u] = max(0, min(left - u * kPageRows, kPageRows));
                    }
                    if constexpr (SCORES == Scores::kNear) {
                        float* const to_scores = near + r0 * G + kPageRows * col + 4 * (lane >> 4);
                        O::attend(st, t[d], from, to, lds, lane, [&](int u, f32x4 x) {
                            if (col < G) *reinterpret_cast<f32x4*>(to_scores + u * kPageRows * G) = x;
                        });
                    } else if constexpr (SCORES == Scores::kFar) {
                        const auto page_scores = __builtin_amdgcn_make_buffer_rsrc(
                            scores + (int64_t)r0 * G, 0, KT * kPageRows * G * (int)sizeof(float), 0x00020000);
                        O::attend(st, t[d], from, to, lds, lane, [&](int u, f32x4 x) {
                            // (The page's offset not as the scalar one: with a register there, the instruction behind the
                            // store may overwrite the data before they are read.)
                            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), page_scores,
                                                                   score_at + u * kPageRows * G * (int)sizeof(float), 0, 0);
                        });
                    } else {
                        O::attend(st, t[d], from, to, lds, lane, NoScores());
                    }
                }
            }
        }
    }
    if (steps <= 0) O::init(st, raw, a.qscale);
    if constexpr (kPages4<T>) O::finish(st);
}

// Inclusive sum over the lanes of a wave, in registers (row shifts, then each row's last lane to the next rows).
__device__ __forceinline__ unsigned lane_scan(unsigned y) {
    int x = (int)y;
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);
    return (unsigned)(x + __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false));
}

// A workgroup's stretch: part `part` of `parts` of one (sequence, kv head).
struct Stretch {
    int s, h, len;  // len: rows_of
    unsigned part, parts;
};

// The stretch of workgroup w where the lengths decide: every (sequence, kv head)
// gets a workgroup for each `share` of its steps, the share being such that the
// workgroups there are suffice.  64 sequences at a time, one a lane; s < 0: no work.
// (Even runs over all steps, whatever sequence they lie in, cost a start and a merge
// more in many workgroups: 128 sequences of 1,024 4-bit rows 17 us instead of 8.)
__device__ __forceinline__ Stretch rows_deal(const RowsArgs& a, unsigned w, int lane) {
    constexpr int C = 4;  // chunks whose lengths are loaded together
    const unsigned kv = a.n_kv_head;
    int len[C];
    auto load = [&](int s0) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int i = s0 + 64 * c + lane;
            len[c] = i < a.n_seq ? rows_of(a, i) : 0;
        }
    };
    auto steps_of = [](int rows) { return ((unsigned)max(rows, 0) + kRowsStep - 1) / kRowsStep; };
    unsigned all = 0;
    load(0);
    for (int s0 = 0;;) {
        unsigned x = 0;
#pragma unroll
        for (int c = 0; c < C; ++c) x += steps_of(len[c]);
        all += (unsigned)__builtin_amdgcn_readlane((int)lane_scan(x), 63);
        s0 += 64 * C;
        if (s0 >= a.n_seq) break;
        load(s0);
    }
    const unsigned spare = a.workgroups - (unsigned)a.n_seq * kv;
    const unsigned share = max((unsigned)kRowsShare, (all * kv + spare - 1) / spare);
    if (a.n_seq > 64 * C) load(0);
    unsigned before = 0;
    for (int s0 = 0;;) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (s0 + 64 * c >= a.n_seq) break;
            const int i = s0 + 64 * c + lane;
            const unsigned parts = max(1u, (steps_of(len[c]) + share - 1) / share), n = i < a.n_seq ? parts * kv : 0;
            const unsigned incl = before + lane_scan(n);
            const uint64_t b = __ballot(incl > w);
            if (b) {
                const int l = __builtin_ctzll(b);
                Stretch r;
                r.s = s0 + 64 * c + l;
                r.len = __builtin_amdgcn_readlane(len[c], l);
                r.parts = (unsigned)__builtin_amdgcn_readlane((int)parts, l);
                const unsigned at = w - (unsigned)__builtin_amdgcn_readlane((int)(incl - n), l);
                r.h = (int)(unsigned)__builtin_amdgcn_readfirstlane((int)(at / r.parts));
                r.part = at - (unsigned)r.h * r.parts;
                return r;
            }
            before = (unsigned)__builtin_amdgcn_readlane((int)incl, 63);
        }
        s0 += 64 * C;
        if (s0 >= a.n_seq) return Stretch{-1, 0, 0, 0, 0};
        load(s0);
    }
}

// One over a head's sum; without a row that takes part (all scores -infinity) the head gives none, as its output.
__device__ __forceinline__ float over_sum(float l) { return l == 0.f ? 0.f : 1.0f / l; }
// Adds a head's weights of four rows: its scores x, its maximum, one over its sum.
__device__ __forceinline__ void add_weights(f32x4& w, f32x4 x, float m, float r) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] += fast_exp2(x[i] - m) * r;
}
__device__ __forceinline__ void put_weights(const RowsArgs& a, int sk, int64_t row, int len, f32x4 w) {
    const int64_t at = (int64_t)sk * a.weight_stride + row;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (row + i < len) a.weights_out[at + i] = (a.weights_in ? a.weights_in[at + i] : 0.f) + w[i];
}

// The weights of four rows, summed over the heads; head g's maximum and one over
// its sum in m and r.  Scores lie by page, head and row: what a step writes and a
// thread reads is close together (by head and row, power-of-two strides apart, 128
// sequences of 8,192 bf16 rows 130 us instead of 125).  Four heads' scores read at
// once took up to 3% longer.
__device__ __forceinline__ void row_weights(const RowsArgs& a, const float* scores, int sk, int64_t row, int len,
                                            const float* m, const float* r) {
    scores += (row & -kPageRows) * a.group + (row & (kPageRows - 1));
    f32x4 w = {0.f, 0.f, 0.f, 0.f};
    for (int g = 0; g < a.group; ++g) add_weights(w, *reinterpret_cast<const f32x4*>(scores + kPageRows * g), m[g], r[g]);
    put_weights(a, sk, row, len, w);
}

template <typename T, int NW>
__device__ __forceinline__ void rows_body(const RowsArgs& a) {
    __shared__ OwnLds<T, NW> lds;
    __shared__ float s_m[kMaxGroupHeads], s_r[kMaxGroupHeads];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int w = blockIdx.x, G = a.group;
    Stretch r;
    if (a.workgroups) {
        r = rows_deal(a, (unsigned)w, lane);
        if (r.s < 0) return;
    } else {
        r.s = w / a.n_kv_head;
        r.h = w - r.s * a.n_kv_head;
        r.len = rows_of(a, r.s);
        r.part = 0;
        r.parts = 1;
    }
    const int sk = r.s * a.n_kv_head + r.h;
    float* out = a.out + (int64_t)sk * G * kHeadDim;
    if (a.workgroups && r.part == 0 && threadIdx.x == 0) {
        a.meta[2 * (size_t)sk] = w;
        a.meta[2 * (size_t)sk + 1] = (int)r.parts;
    }
    if (r.len <= 0) {  // zeros, or NaN for a length that the launch does not cover
        if (r.len < 0 && threadIdx.x == 0) atomicOr(a.err, 2);
        for (int i = threadIdx.x; i < G * kHeadDim; i += 64 * NW) out[i] = r.len < 0 ? __builtin_nanf("") : 0.f;
        return;
    }
    const bool whole = r.parts == 1;
    int lo = 0, hi = r.len;
    if (!whole) {  // (the last parts may be shorter, or empty)
        const unsigned per = (((unsigned)r.len + kRowsStep - 1) / kRowsStep + r.parts - 1) / r.parts * kRowsStep;
        lo = (int)min((unsigned)r.len, r.part * per);
        hi = (int)min((unsigned)r.len, lo + per);
    }
    typename Own<T>::State st;
    extern __shared__ f32x4 near4[];
    float* const near = reinterpret_cast<float*>(near4);
    if (a.near)
        rows_attend<T, NW, Scores::kNear>(a, st, lds.own[wave], r.s, r.h, lo, hi, wave, lane, near);
    else if (a.scores)
        rows_attend<T, NW, Scores::kFar>(a, st, lds.own[wave], r.s, r.h, lo, hi, wave, lane, near);
    else
        rows_attend<T, NW, Scores::kNone>(a, st, lds.own[wave], r.s, r.h, lo, hi, wave, lane, near);
    merge_waves<T, NW>(st, lds.merge, wave, lane, [&](int c, int d, float M, float L, f32x4 A) {
        if (c >= G) return;
        const size_t p = (size_t)w * G + c;
        if (whole)
            *reinterpret_cast<f32x4*>(out + c * kHeadDim + d) = finish_row(A, L);
        else
            *reinterpret_cast<f32x4*>(a.part + p * kHeadDim + d) = A;
        if (d == 0 && !whole) *reinterpret_cast<float2*>(a.ml + 2 * p) = make_float2(M, L);
        if (d == 0 && whole) {
            s_m[c] = M;
            s_r[c] = over_sum(L);
        }
    });
    if (!whole || !a.weights_out) return;
    __syncthreads();  // all scores and sums are there
    if (a.near) {
        for (int row = 4 * (int)threadIdx.x; row < r.len; row += 4 * 64 * NW)
            row_weights(a, near, sk, row, r.len, s_m, s_r);
    } else {
        const float* scores = a.scores + (int64_t)sk * G * a.score_stride;
        for (int64_t row = 4 * (int)threadIdx.x; row < r.len; row += 4 * 64 * NW)
            row_weights(a, scores, sk, row, r.len, s_m, s_r);
    }
}

// What follows where sequences are cut: of every (sequence, kv head) of several
// workgroups, merge_blocks workgroups merge the partials, a head a wave or, where there
// are as many workgroups as heads, a head all four; the others take the weights of
// 1,024 rows each: a head's maximum and sum from the partials, 16 lanes a head, then
// four rows a thread, summed over the heads, whose scores are under way before that.
// A launch and the chain partials -> maximum: 3.2 us without weights, 6 with those of
// 64 sequences of up to 4,096 rows (18 MB; scores read after the maxima: 0.3 more, 0.5
// at one of 2,000).
template <int WPR>
__device__ __forceinline__ void merge_parts(const RowsArgs& a, int64_t row, int c, int p0, int n, int w, int lane) {
    constexpr int kRound = 16 * WPR;
    const int sub = lane >> 4, G = a.group;
    const float* acc = a.part + ((size_t)p0 * G + c) * kHeadDim + 4 * (lane & 15);
    const float2* ml = reinterpret_cast<const float2*>(a.ml) + (size_t)p0 * G + c;
    float M = kNoMax, L = 0.f;
    f32x4 A = {0.f, 0.f, 0.f, 0.f};
    for (int c0 = 0; c0 < n; c0 += kRound) {
        f32x4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = c0 + 4 * (WPR * i + w) + sub;
            v[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (e < n) v[i] = *reinterpret_cast<const f32x4*>(acc + (size_t)e * G * kHeadDim);
        }
        float2 x = make_float2(kNoMax, 0.f);
        if (lane < kRound && c0 + lane < n) x = ml[(size_t)(c0 + lane) * G];
        const float m1 = fmaxf(M, xor_max<1>(x.x));
        const float f = fast_exp2(M - m1), y = fast_exp2(x.x - m1);
        L = L * f + xor_sum<1>(x.y * y);
        A *= f;
        M = m1;
#pragma unroll
        for (int i = 0; i < 4; ++i) A += __shfl(y, (4 * (WPR * i + w) + sub) & 63) * v[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) A[i] = xor_sum<16>(A[i]);
    if constexpr (WPR > 1) {
        __shared__ f32x4 s_a[WPR][16];
        if (lane < 16) s_a[w][lane] = A;
        __syncthreads();
        if (lane < 16) {
            A = s_a[0][lane];
#pragma unroll
            for (int i = 1; i < WPR; ++i) A += s_a[i][lane];
        }
    }
    if (w == 0 && lane < 16) *reinterpret_cast<f32x4*>(a.out + row * kHeadDim + 4 * lane) = finish_row(A, L);
}

__device__ __forceinline__ void rows_finish_body(const RowsArgs& a) {
    __shared__ float s_m[kMaxGroupHeads], s_r[kMaxGroupHeads];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), G = a.group;
    const int per = a.merge_blocks + a.weight_blocks;
    const int sk = blockIdx.x / per, i0 = blockIdx.x - sk * per, s = sk / a.n_kv_head, h = sk - s * a.n_kv_head;
    const int64_t row0 = (int64_t)s * a.n_head + h * G;
    const int len = rows_of(a, s), p0 = a.meta[2 * (size_t)sk], n = a.meta[2 * (size_t)sk + 1];
    if (len <= 0 || n == 1) return;  // its workgroup did it all
    if (i0 < a.merge_blocks) {
        if (a.merge_blocks == G) {
            merge_parts<kPagedWaves>(a, row0 + i0, i0, p0, n, wave, lane);
        } else {
            for (int c = i0 * kPagedWaves + wave; c < G; c += kPagedWaves * a.merge_blocks)
                merge_parts<1>(a, row0 + c, c, p0, n, 0, lane);
        }
        return;
    }
    const int64_t block0 = (int64_t)(i0 - a.merge_blocks) * 1024, row = block0 + 4 * tid;
    if (block0 >= len) return;
    // The first heads' scores are on their way while the maxima are joined.
    constexpr int kFirst = 8;
    const int64_t at = min(row, (int64_t)(len - 1) & -4);
    const float* const scores = a.scores + (int64_t)sk * G * a.score_stride + (at & -kPageRows) * G + (at & (kPageRows - 1));
    f32x4 y[kFirst];
#pragma unroll
    for (int g = 0; g < kFirst; ++g) y[g] = *reinterpret_cast<const f32x4*>(scores + kPageRows * min(g, G - 1));
    const float2* ml = reinterpret_cast<const float2*>(a.ml) + (size_t)p0 * G;
    const int c = tid >> 4, sub = tid & 15;
    if (c < G) {
        float m = kNoMax, l = 0.f;
        for (int i = sub; i < n; i += 16) {
            const float2 x = ml[(size_t)i * G + c];
            const float m1 = fmaxf(m, x.x);
            l = l * fast_exp2(m - m1) + x.y * fast_exp2(x.x - m1);
            m = m1;
        }
#pragma unroll
        for (int i = 1; i < 16; i *= 2) {
            const float m2 = __shfl_xor(m, i), l2 = __shfl_xor(l, i), m1 = fmaxf(m, m2);
            l = l * fast_exp2(m - m1) + l2 * fast_exp2(m2 - m1);
            m = m1;
        }
        if (sub == 0) {
            s_m[c] = m;
            s_r[c] = over_sum(l);
        }
    }
    __syncthreads();
    if (row >= len) return;
    f32x4 w = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < kFirst; ++g) {
        if (g >= G) break;
        add_weights(w, y[g], s_m[g], s_r[g]);
    }
    for (int g = kFirst; g < G; ++g)
        add_weights(w, *reinterpret_cast<const f32x4*>(scores + kPageRows * g), s_m[g], s_r[g]);
    put_weights(a, sk, row, len, w);
}

// ---------------------------------------------------------------------------
// Rows to keep.  One workgroup a (sequence, kv head).  The keep-th largest key
// (the weights' bits in order, the first and last rows above all) is found
// eleven bits at a time: a histogram in LDS of the digits of the keys that agree
// with the bits found so far, and the digit at which its sum from the top passes
// what is left; a digit all of whose keys are kept ends the search.  Then every
// wave counts, and places, the rows of its own run: those above the key, and the
// first of those equal to it.  Up to three rounds over the keys in registers, each a
// chain of counts and barriers, bound it, not the bytes: 2 lists of 2,048 take 5.7 us
// (3 of them the launch), 128 of 8,192 to 16,384 14.7, on half the CUs.  (The
// first form, 1,024 threads and no early end: 8.1 and 17.9.)
constexpr int kRowsBins = 2048;
template <int NT, int REGS>  // threads; keys a thread holds, of longer lists it reads the rest again
__device__ __forceinline__ void select_rows_body(const SelectRowsArgs& a) {
    constexpr int NW = NT / 64, PER = kRowsBins / NT;
    __shared__ unsigned s_bin[kRowsBins];
    __shared__ unsigned s_sum[16], s_eq[16];
    __shared__ unsigned s_found[3];  // digit, keys above it, keys of it
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int sk = blockIdx.x, s = sk / a.n_kv_head;
    const int len = max(a.lengths[s], 0), n = len > a.max_len ? 0 : len;
    int32_t* out = a.kept + (size_t)sk * a.keep;
    if (len > a.max_len && tid == 0) atomicOr(a.err, 2);
    if (n <= a.keep) {
        for (int i = tid; i < a.keep; i += NT) out[i] = i < n ? i : -1;
        return;
    }
    const float* w = a.weights + sk * a.weight_stride;
    const int rounds = (n + NT - 1) / NT, j0 = wave * rounds * 64 + lane;  // this lane's: j0 + 64 r
    auto key_at = [&](int r) {  // 0: behind the last row (no weight has that key)
        const int64_t j = (int64_t)j0 + 64 * (int64_t)r;
        return j >= n ? 0u : j < a.first || j >= n - a.last ? 0xFFFFFFFFu : order_key(w[j]);
    };
    unsigned k[REGS];
#pragma unroll
    for (int r = 0; r < REGS; ++r) k[r] = r < rounds ? key_at(r) : 0u;
    auto each = [&](auto f) {
#pragma unroll
        for (int r = 0; r < REGS; ++r)
            if (r < rounds) f(k[r], r);
        for (int r = REGS; r < rounds; ++r) f(key_at(r), r);
    };
    // what the waves before this one left in sums, and this lane's place in its wave
    auto of_waves_before = [&](const unsigned* sums) {
        const unsigned x = lane_scan(lane < NW ? sums[lane & 15] : 0u);
        return wave ? (unsigned)__builtin_amdgcn_readlane((int)x, wave - 1) : 0u;
    };
    auto lanes_before = [](uint64_t b) {
        return __builtin_amdgcn_mbcnt_hi((unsigned)(b >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)b, 0u));
    };
    unsigned prefix = 0, mask = 0, left = (unsigned)a.keep;  // of the keys with key & mask == prefix the left largest are kept
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const unsigned digits = pass == 2 ? 1023u : 2047u;
#pragma unroll
        for (int i = 0; i < PER; ++i) s_bin[tid + i * NT] = 0;
        __syncthreads();
        each([&](unsigned x, int) {
            if (x && (x & mask) == prefix) atomicAdd(&s_bin[x >> shift & digits], 1u);
        });
        __syncthreads();
        // PER bins a thread, from the top
        unsigned c[PER], sum = 0;
        const int top = kRowsBins - 1 - PER * tid;
#pragma unroll
        for (int i = 0; i < PER; ++i) sum += c[i] = s_bin[top - i];
        const unsigned incl = lane_scan(sum);
        if (lane == 63) s_sum[wave] = incl;
        __syncthreads();
        unsigned before = of_waves_before(s_sum) + incl - sum;
        if (before < left && before + sum >= left) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if (before < left && before + c[i] >= left) {
                    s_found[0] = (unsigned)(top - i);
                    s_found[1] = before;
                    s_found[2] = c[i];
                }
                before += c[i];
            }
        }
        __syncthreads();
        prefix |= s_found[0] << shift;
        left -= s_found[1];
        mask |= digits << shift;
        if (left == s_found[2] && prefix) {  // all of them: the keys above the one below
            --prefix;
            left = 0;
            break;
        }
    }
    // keys above prefix are kept, and the first `left` of those equal to it
    unsigned gt = 0, eq = 0;
    each([&](unsigned x, int) {
        gt += __popcll(__ballot(x > prefix));
        eq += __popcll(__ballot(x == prefix));
    });
    if (lane == 0) {
        s_sum[wave] = gt;
        s_eq[wave] = eq;
    }
    __syncthreads();
    gt = of_waves_before(s_sum);
    eq = of_waves_before(s_eq);
    int32_t* o = out + gt + min(eq, left);  // the next row's place
    each([&](unsigned x, int r) {
        uint64_t b = __ballot(x > prefix);
        if (eq < left) {
            const uint64_t be = __ballot(x == prefix);
            if (be) {
                b |= __ballot(x == prefix && eq + lanes_before(be) < left);
                eq += __popcll(be);
            }
        }
        if (b >> lane & 1) o[lanes_before(b)] = j0 + 64 * r;
        o += __popcll(b);
    });
}

// ---------------------------------------------------------------------------
// Compaction: a copy through a list, bound by memory.  A wave takes 16 kept rows
// of one (sequence, kv head), the rows of one destination page.  The chain list
// -> table -> row is three loads deep, so a wave has all of its page's rows in
// flight at once, two to eight 16-byte loads a lane, and no barrier.  Loads are
// unconditional (a place without a row reads another's row), stores are not.
// 40 sequences of up to 8,001 rows kept to 4,001, 2 kv heads, from memory: bf16
// 168 MB 40.6 us (4.1 TB/s), fp32 74, Q8_0 41, 4-bit 28 (rows of 68 and 36 bytes lie
// across lines of 128).  Four lanes' worth of loads less a wave and barriers: 50, 77,
// 69 and 55.
template <typename T>
__device__ __forceinline__ void compact_body(const CompactArgs& a) {
    const int lane = threadIdx.x & 63, kv = a.n_kv_head;
    // kv heads next to each other: the ends of their rows share lines
    const int unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sp = unit / kv, h = unit - sp * kv, s = sp / a.n_grid, jp = sp - s * a.n_grid;
    if (s >= a.n_seq) return;
    const int64_t sk = (int64_t)s * kv + h;
    // Lanes 0..15 (and their copies): source page of the pool * 16 + row in it, -1: no row.
    const int j = jp * kPageRows + (lane & 15);
    const int row = j < a.keep ? a.kept[sk * a.keep + j] : -1;
    // (a list may be wider than its destination: its places past to_pages have no page)
    const int to = jp < a.to_pages ? a.to_table[(size_t)s * a.to_pages + jp] : -1, len = a.lengths[s];
    int64_t src = -1;
    float weight = 0.f;
    bool bad = false;
    if (row >= 0 && row < len && row < (int64_t)a.max_pages * kPageRows && (!a.weights_out || max(row, j) < a.weight_stride)) {
        const int page = a.block_table[(size_t)s * a.max_pages + (row >> kPageShift)];
        if (a.weights_out) weight = a.weights_in[sk * a.weight_stride + row];
        bad = page < 0 || page >= a.n_pages;
        src = (int64_t)min(max(page, 0), a.n_pages - 1) * kPageRows + (row & (kPageRows - 1));
    } else {
        bad = row != -1;
    }
    const unsigned rows = (unsigned)__ballot(src >= 0) & 0xffff;
    const bool to_bad = to < 0 || to >= a.n_pages;
    if ((__any(bad) || (rows && to_bad)) && lane == 0) atomicOr(a.err, 4);
    const auto weights = [&]() {  // behind the rows' loads
        if (!a.weights_out) return;
        float* const out = a.weights_out + sk * a.weight_stride;
        const int64_t listed = min((int64_t)a.keep, a.weight_stride);
        if (lane < 16 && j < listed) out[j] = weight;
        // what follows the last kept row, shared out among the pages' waves
        const int64_t part = (a.weight_stride - listed + a.n_grid - 1) / a.n_grid, b = listed + jp * part;
        const int64_t e = min(b + part, a.weight_stride);
        for (int64_t i = b + lane; i < e; i += 64) out[i] = 0.f;
    };
    if (!rows || to_bad) return weights();
    const int64_t other = __shfl(src, __builtin_ctz(rows));
    src = src < 0 ? other : src;
    const size_t page_bytes = PageFmt<T>::page(kv), head = PageFmt<T>::head(h);
    char* const pools[2] = {a.k_pages, a.v_pages};
    if constexpr (__is_same(T, q4_t)) {
        // Of k, lane (g, r) moves the 8 bytes of row r's dims 16 g ..  Of v, 16 lanes a quad of rows: lane i has the
        // quad's dims i + 16 d, a byte of 8 for each row, taken from the byte of each source row that is its place there.
        const int r = lane & 15, g = lane >> 4;
        const int r1 = (int)src & (kPageRows - 1);
        const char* from = a.k_pages + (src >> kPageShift) * page_bytes + head;
        const u32x2 k = *reinterpret_cast<const u32x2*>(from + 8 * (16 * g + r1));
        const uint16_t kd = reinterpret_cast<const uint16_t*>(from)[256 + 16 * (g & 1) + r1];
        const auto place = [](int x) { return (x & 3) == 1 ? 2 : (x & 3) == 2 ? 1 : x & 3; };
        u32x2 v[4];
        uint16_t vd[4];
        int at[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int64_t sq = __shfl(src, 4 * g + q);
            at[q] = (int)sq & (kPageRows - 1);
            const char* vf = a.v_pages + (sq >> kPageShift) * page_bytes + head;
            v[q] = *reinterpret_cast<const u32x2*>(vf + 8 * (16 * (at[q] >> 2) + r));
            vd[q] = reinterpret_cast<const uint16_t*>(vf)[256 + 8 * (at[q] >> 2) + 4 * (r & 1) + (at[q] & 3)];
        }
        weights();
        char* const kt = a.k_pages + (size_t)to * page_bytes + head;
        char* const vt = a.v_pages + (size_t)to * page_bytes + head;
        if (rows >> r & 1) {
            *reinterpret_cast<u32x2*>(kt + 8 * (16 * g + r)) = k;
            if (g < 2) reinterpret_cast<uint16_t*>(kt)[256 + 16 * g + r] = kd;
        }
        const unsigned quad = rows >> (4 * g) & 15;
        u32x2* const vo = reinterpret_cast<u32x2*>(vt + 8 * (16 * g + r));
        u32x2 w = {0, 0};
        if (quad && quad != 15) w = *vo;  // rows without a source stay
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (!(quad >> q & 1)) continue;
            const int to8 = 8 * place(q), at8 = 8 * place(at[q]);
#pragma unroll
            for (int p = 0; p < 2; ++p) w[p] = (w[p] & ~(0xffu << to8)) | ((v[q][p] >> at8 & 0xff) << to8);
            if (r < 2) reinterpret_cast<uint16_t*>(vt)[256 + 8 * g + 4 * r + q] = vd[q];
        }
        if (quad) *vo = w;
    } else {
        // LANES lanes a row, 16 bytes each; rows of 68 bytes have another four.
        constexpr int HB = CacheFmt<T>::kHeadBytes, LANES = HB / 16, STEPS = kPageRows * LANES / 64;
        constexpr bool TAIL = HB % 16 != 0;
        static_assert(HB == 16 * LANES + 4 * TAIL && (LANES == 4 || !TAIL), "whole steps");
        const size_t row_bytes = PageFmt<T>::row(kv);
        const int r0 = lane / LANES, c = lane % LANES;
        u32x4_a4 x[2][STEPS];
        unsigned tail[2];
#pragma unroll
        for (int t = 0; t < STEPS; ++t) {
            const int64_t sr = __shfl(src, r0 + t * (64 / LANES));
            const size_t off = (sr >> kPageShift) * page_bytes + (sr & (kPageRows - 1)) * row_bytes + head;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                x[v][t] = *reinterpret_cast<const u32x4_a4*>(pools[v] + off + 16 * c);
                if constexpr (TAIL) tail[v] = *reinterpret_cast<const unsigned*>(pools[v] + off + 16 * LANES);
            }
        }
        weights();
#pragma unroll
        for (int t = 0; t < STEPS; ++t) {
            const int r = r0 + t * (64 / LANES);
            if (!(rows >> r & 1)) continue;
            const size_t off = (size_t)to * page_bytes + r * row_bytes + head;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                *reinterpret_cast<u32x4_a4*>(pools[v] + off + 16 * c) = x[v][t];
                if constexpr (TAIL)
                    if (c == 0) *reinterpret_cast<unsigned*>(pools[v] + off + 16 * LANES) = tail[v];
            }
        }
    }
}
