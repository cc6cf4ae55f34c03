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
// row of K (first half of the slots) or V.
template <typename T>
__device__ __forceinline__ void widen_body(const WidenArgs& a) {
    const int c = threadIdx.x & 7, r = threadIdx.x >> 3 & 15, v = threadIdx.x >> 7;
    if (!a.pages[v]) return;
    const int64_t unit = blockIdx.x;
    const int page = (int)(unit / a.n_kv_head), h = (int)(unit - (int64_t)page * a.n_kv_head);
    const char* p = a.pages[v] + (size_t)page * PageFmt<T>::page(a.n_kv_head) + PageFmt<T>::head(h);
    float x[8];
    if constexpr (__is_same(T, q4_t))
        load_row4(x, p, r, c, v == 0);
    else
        load_row<T, false>(x, p + r * PageFmt<T>::row(a.n_kv_head) + 4 * c * CacheFmt<T>::kDimBytes, c);
    store8(a.out[v] + (((size_t)page * kPageRows + r) * a.n_kv_head + h) * kHeadDim + 4 * c, x);
}

// ---------------------------------------------------------------------------
// Append at given rows.  The rows' sequences are found as in append_body; a
// pair (d, d + 1) turns by the position on its axis, so a lane reads the four
// (cos, sin) of its pairs from up to four table rows.
template <typename T>
__device__ __forceinline__ void append_axes_body(const AppendAxesArgs& x_args) {
    const AppendArgs& a = x_args.a;
    __shared__ int s_seq[kAppendRows];
    __shared__ int64_t s_page[kAppendRows];  // pool page, -1: not stored
    __shared__ int s_at[kAppendRows];        // row in the page, -1: the row is skipped
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
            for (int i = 0; i < x_args.n_axes; ++i)
                ok &= (unsigned)x_args.pos[(size_t)i * a.n_rows + t0 + tid] < (unsigned)x_args.max_pos;
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
    const int nh = a.q ? a.n_head : 0, kv = a.n_kv_head, per = nh + 2 * kv;
    for (int it = slot; it < n * per; it += 32) {
        const int r = it / per, h = it - r * per, at = s_at[r];
        if (at < 0) continue;
        const int64_t t = t0 + r, page = s_page[r];
        float x[8];
        auto turn = [&]() {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int pair = (i < 2 ? 0 : 16) + 2 * c + (i & 1);
                const int axis = (int)(x_args.pair_axis >> (2 * pair)) & 3;
                const float2 cs = a.rope_cs[(size_t)x_args.pos[(size_t)axis * a.n_rows + t] * (kHeadDim / 2) + pair];
                rotate_pair(x[2 * i], x[2 * i + 1], cs.x, cs.y);
            }
        };
        if (h < nh) {
            load8(x, a.q + t * a.q_stride + (int64_t)h * kHeadDim + 4 * c);
            turn();
            store8(a.q_out + (t * nh + h) * kHeadDim + 4 * c, x);
        } else if (page >= 0) {
            const bool key = h < nh + kv;
            const int hk = key ? h - nh : h - nh - kv;
            load8(x, (key ? a.k + t * a.k_stride : a.v + t * a.v_stride) + (int64_t)hk * kHeadDim + 4 * c);
            if (key) turn();
            char* p = (key ? a.k_pages : a.v_pages) + (size_t)page * PageFmt<T>::page(kv) + PageFmt<T>::head(hk);
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
// subtraction and a product with the scale (a sixteenth of it) the pair of
// values, all exact.
template <>
struct Own<q4_t> {
    using S = Mfma16;
    using State = Cols<_Float16, S>;
    using RawQuery = RawQ<_Float16, S>;
    static constexpr int kTiles = 2;
    struct Tile {
        u32x2 k, v;
        unsigned kd;  // scale of row lane % 16, dims 16 (lane / 16) ..
        u32x4 vd;     // scales of rows 4 (lane / 16) .. of dims 0 .. 31, then 32 .. 63
    };
    struct Lds {};
    // Dims 16 g + 8 m + 0..7: the operand of product m.
    __device__ static void query(RawQuery& q, const float* p, int lane) {
        const int g = lane >> 4;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                q.x[m][i] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (p) q.x[m][i] = *reinterpret_cast<const f32x4*>(p + 16 * g + 8 * m + 4 * i);
            }
    }
    __device__ static void init(State& st, const RawQuery& q, float scale) { cols_init<_Float16, S>(st, q, scale); }
    __device__ static void fetch(Tile& t, const char* kp, const char* vp, size_t, int lane) {
        const int i = lane & 15, g = lane >> 4;
        t.k = *reinterpret_cast<const u32x2*>(kp + 8 * lane);
        t.v = *reinterpret_cast<const u32x2*>(vp + 8 * lane);
        t.kd = *reinterpret_cast<const uint16_t*>(kp + 512 + 32 * (g >> 1) + 2 * i);
        t.vd = *reinterpret_cast<const u32x4*>(vp + 512 + 16 * g);
    }
    __device__ static f16x2 low(unsigned w) {
        const f16x2 bias = {(_Float16)1032.0f, (_Float16)1032.0f};
        return __builtin_bit_cast(f16x2, (w & 0x000F000Fu) | 0x64006400u) - bias;
    }
    __device__ static f16x2 high(unsigned w) {
        const f16x2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
        return __builtin_bit_cast(f16x2, (w & 0x00F000F0u) | 0x64006400u) - bias;
    }
    static constexpr _Float16 kSixteenth = (_Float16)0.0625f;
    // Keys lo[u] .. hi[u] - 1 of page u take part.
    template <typename Score>
    __device__ static void attend(State& st, const Tile (&t)[kTiles], const int (&lo)[kTiles], const int (&hi)[kTiles],
                                  Lds&, int lane, Score score) {
        using M = MMath<_Float16>;
        const int g = lane >> 4;
        const bool full = lo[0] <= 0 && lo[1] <= 0 && hi[0] >= kPageRows && hi[1] >= kPageRows;
        f32x4 w[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const _Float16 d = __builtin_bit_cast(_Float16, (unsigned short)t[u].kd);
            const f16x2 d0 = {d, d}, d1 = d0 * f16x2{kSixteenth, kSixteenth};
            w[u] = score_tile<_Float16, S>(st, nullptr, nullptr, g, [&](int m, int) {
                const unsigned x = t[u].k[m], y = x >> 8;
                const f16x2 e[4] = {low(x) * d0, high(x) * d1, low(y) * d0, high(y) * d1};
                return __builtin_bit_cast(M::v8, e);
            });
        }
        u32x4 vd[2] = {t[0].vd, t[1].vd};
        if (!full) {
            asm volatile("");  // a branch, not selects
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                auto in = [&](int r) { return 4 * g + r >= lo[u] && 4 * g + r < hi[u]; };
#pragma unroll
                for (int r = 0; r < 4; ++r) w[u][r] = in(r) ? w[u][r] : kNegInf;
                // a row outside may hold any scale
                const unsigned m0 = (in(0) ? 0xFFFFu : 0u) | (in(1) ? 0xFFFF0000u : 0u);
                const unsigned m1 = (in(2) ? 0xFFFFu : 0u) | (in(3) ? 0xFFFF0000u : 0u);
                vd[u] = u32x4{vd[u][0] & m0, vd[u][1] & m1, vd[u][2] & m0, vd[u][3] & m1};
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) score(u, w[u] + st.base);
        softmax_step<S>(st.m, st.l, st.base, st.o, w);
        M::v8 px[2];
        {
            u32x4 p[2];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    unsigned z[3] = {0, 0, 0};
                    split<M, 2>(w[u][2 * r] * M::kPScale, w[u][2 * r + 1] * M::kPScale, z);
                    p[0][2 * u + r] = z[0];
                    p[1][2 * u + r] = z[1];
                }
#pragma unroll
            for (int i = 0; i < 2; ++i) px[i] = __builtin_bit_cast(M::v8, p[i]);
        }
#pragma unroll
        for (int p = 0; p < 2; ++p) {  // dims 32 p + i, then 32 p + 16 + i
            f16x2 e[2][4];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const unsigned x = t[u].v[p], y = x >> 8;
                // (a copy first: the bit cast of a vector's element reads the vector's first one)
                const unsigned a0 = vd[u][2 * p], b0 = vd[u][2 * p + 1];
                const f16x2 a = __builtin_bit_cast(f16x2, a0), b = __builtin_bit_cast(f16x2, b0);
                const f16x2 s = {kSixteenth, kSixteenth};
                e[0][2 * u] = low(x) * a;
                e[0][2 * u + 1] = low(y) * b;
                e[1][2 * u] = high(x) * (a * s);
                e[1][2 * u + 1] = high(y) * (b * s);
            }
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    st.o[2 * p + b] = M::mfma32(__builtin_bit_cast(M::v8, e[b]), px[i], st.o[2 * p + b]);
        }
    }
    static constexpr int dim(int b, int g) { return 16 * b + 4 * g; }
    __device__ static f32x4 sums(const State& st, int b) { return st.o[b] * (1.0f / MMath<_Float16>::kPScale); }
};

// ---------------------------------------------------------------------------
// Attention over whole sequences: workgroup (slot of slot_rows rows, kv head,
// sequence).  With a.scores set it leaves every score, and the slot's (m, l)
// also where it is the only one, for the weights.
template <typename T, int NW>
__device__ __forceinline__ void rows_body(const PagedAttnArgs& a) {
    __shared__ OwnLds<T, NW> lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kv = a.n_kv_head, G = a.group;
    const int split = blockIdx.x % a.n_slots, sk = blockIdx.x / a.n_slots, s = sk / kv, h = sk - s * kv;
    const int len = max(a.lengths[s], 0);
    const bool bad = len > a.max_len;
    const int64_t lo = (int64_t)split * a.slot_rows, hi = bad ? lo : min((int64_t)len, lo + a.slot_rows);
    const int64_t row0 = (int64_t)s * a.n_head + h * G;
    const int col = lane & 15;
    typename Own<T>::RawQuery raw;
    typename Own<T>::State st;
    Own<T>::query(raw, col < G ? a.q + (row0 + col) * kHeadDim : nullptr, lane);
    Own<T>::init(st, raw, a.qscale);
    if (lo < hi) {
        const int j0 = (int)(lo >> kPageShift), n = (int)((hi - 1) >> kPageShift) - j0 + 1;
        const int32_t* table = a.block_table + (size_t)s * a.max_pages;
        float* scores = a.scores && col < G ? a.scores + (row0 + col) * a.score_stride + 4 * (lane >> 4) : nullptr;
        attend_run<T, NW>(
            st, a, h, n, lo, hi, lds.own[wave], wave, lane,
            [&](int e, int& logical, int& page) {
                logical = j0 + e;
                page = table[logical];
                if (page < 0 || page >= a.n_pages) {
                    atomicOr(a.err, 4);
                    page = min(max(page, 0), a.n_pages - 1);
                }
            },
            [&](int j, f32x4 x) {
                if (scores && j >= 0) *reinterpret_cast<f32x4*>(scores + (int64_t)j * kPageRows) = x;
            });
    }
    merge_waves<T, NW>(st, lds.merge, wave, lane, [&](int c, int d, float M, float L, f32x4 A) {
        if (c >= G) return;
        if (bad) {
            if (split == 0 && c == 0 && d == 0) atomicOr(a.err, 2);
            const float nan = __builtin_nanf("");
            L = nan;
            A = f32x4{nan, nan, nan, nan};
        }
        if (a.n_slots == 1) *reinterpret_cast<f32x4*>(a.out + (row0 + c) * kHeadDim + d) = finish_row(A, L);
        if (a.n_slots > 1 || a.scores) put_partial(a, row0 + c, split, d, M, L, A);
    });
}

// Weights of the rows: workgroup (1,024 rows, (sequence, kv head)).  A head's
// maximum and sum come from the slots' partials, 16 lanes a head; then a thread
// takes four rows and adds their weights over the heads.
__device__ __forceinline__ void row_weights_body(const PagedAttnArgs& a) {
    __shared__ float s_m[kMaxGroupHeads], s_r[kMaxGroupHeads];
    const int tid = threadIdx.x, sk = blockIdx.y, s = sk / a.n_kv_head, h = sk - s * a.n_kv_head, G = a.group;
    const int len = max(a.lengths[s], 0);
    const int64_t row = 4 * ((int64_t)blockIdx.x * 256 + tid);
    if ((int64_t)blockIdx.x * 1024 >= len || len > a.max_len) return;
    const int64_t row0 = (int64_t)s * a.n_head + h * G;
    const float2* ml = reinterpret_cast<const float2*>(a.ws + (size_t)a.n_seq * a.n_head * a.n_slots * kHeadDim);
    const int c = tid >> 4, sub = tid & 15;
    if (c < G) {
        float m = kNoMax, l = 0.f;
        for (int i = sub; i < a.n_slots; i += 16) {
            const float2 x = ml[(row0 + c) * a.n_slots + i];
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
            s_r[c] = 1.0f / l;
        }
    }
    __syncthreads();
    if (row >= len) return;
    f32x4 w = {0.f, 0.f, 0.f, 0.f};
    for (int g = 0; g < G; ++g) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(a.scores + (row0 + g) * a.score_stride + row);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] += fast_exp2(x[i] - s_m[g]) * s_r[g];
    }
    const int64_t at = (int64_t)sk * a.weight_stride + row;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (row + i < len) a.weights_out[at + i] = (a.weights_in ? a.weights_in[at + i] : 0.f) + w[i];
}

// ---------------------------------------------------------------------------
// Rows to keep.  One workgroup a (sequence, kv head).  The keep-th largest key
// (the weights' bits in order, the first and last rows above all) is found
// eleven bits at a time: a histogram in LDS of the digits of the keys that agree
// with the bits found so far, and the digit at which its sum from the top passes
// what is left.  Then every wave counts, and places, the rows of its own run: those
// above the key, and the first of those equal to it.
constexpr int kRowsWaves = 16, kRowsThreads = 64 * kRowsWaves, kRowsBins = 2048;
constexpr int kRowsRegs = 16;  // keys a thread holds; of longer lists it reads the rest again
__device__ __forceinline__ void select_rows_body(const SelectRowsArgs& a) {
    __shared__ unsigned s_bin[kRowsBins];
    __shared__ unsigned s_sum[kRowsWaves], s_eq[kRowsWaves];
    __shared__ unsigned s_found[2];  // digit, keys above it
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int sk = blockIdx.x, s = sk / a.n_kv_head;
    const int len = max(a.lengths[s], 0), n = len > a.max_len ? 0 : len;
    int32_t* out = a.kept + (size_t)sk * a.keep;
    if (len > a.max_len && tid == 0) atomicOr(a.err, 2);
    if (n <= a.keep) {
        for (int i = tid; i < a.keep; i += kRowsThreads) out[i] = i < n ? i : -1;
        return;
    }
    const float* w = a.weights + sk * a.weight_stride;
    const int rounds = (n + kRowsThreads - 1) / kRowsThreads, j0 = wave * rounds * 64 + lane;  // this lane's: j0 + 64 r
    auto key_at = [&](int r) {  // 0: behind the last row (no weight has that key)
        const int64_t j = (int64_t)j0 + 64 * (int64_t)r;
        return j >= n ? 0u : j < a.first || j >= n - a.last ? 0xFFFFFFFFu : order_key(w[j]);
    };
    unsigned k[kRowsRegs];
#pragma unroll
    for (int r = 0; r < kRowsRegs; ++r) k[r] = r < rounds ? key_at(r) : 0u;
    unsigned prefix = 0, mask = 0, left = (unsigned)a.keep;  // of the keys with key & mask == prefix the left largest are kept
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
        for (int i = tid; i < kRowsBins; i += kRowsThreads) s_bin[i] = 0;
        __syncthreads();
        auto count = [&](unsigned x) {
            if (x && (x & mask) == prefix) atomicAdd(&s_bin[x >> shift & (unsigned)(bins - 1)], 1u);
        };
#pragma unroll
        for (int r = 0; r < kRowsRegs; ++r) {
            if (r < rounds) count(k[r]);
        }
        for (int r = kRowsRegs; r < rounds; ++r) count(key_at(r));
        __syncthreads();
        // two bins a thread, from the top
        const int b1 = kRowsBins - 1 - 2 * tid;
        const unsigned c1 = s_bin[b1], c0 = s_bin[b1 - 1];
        const unsigned incl = (unsigned)wave_scan((int)(c0 + c1), lane);
        if (lane == 63) s_sum[wave] = incl;
        __syncthreads();
        unsigned before = incl - c0 - c1;
        for (int i = 0; i < wave; ++i) before += s_sum[i];
        if (before < left && before + c0 + c1 >= left) {
            const bool upper = before + c1 >= left;
            s_found[0] = (unsigned)(upper ? b1 : b1 - 1);
            s_found[1] = upper ? before : before + c1;
        }
        __syncthreads();
        prefix |= s_found[0] << shift;
        left -= s_found[1];
        mask |= (unsigned)(bins - 1) << shift;
    }
    // keys above prefix are kept, and the first `left` of those equal to it
    unsigned gt = 0, eq = 0;
    auto tally = [&](unsigned x) {
        gt += __popcll(__ballot(x > prefix));
        eq += __popcll(__ballot(x == prefix));
    };
#pragma unroll
    for (int r = 0; r < kRowsRegs; ++r) {
        if (r < rounds) tally(k[r]);
    }
    for (int r = kRowsRegs; r < rounds; ++r) tally(key_at(r));
    if (lane == 0) {
        s_sum[wave] = gt;
        s_eq[wave] = eq;
    }
    __syncthreads();
    gt = eq = 0;
    for (int i = 0; i < wave; ++i) {
        gt += s_sum[i];
        eq += s_eq[i];
    }
    auto place = [&](unsigned x, int r) {
        const uint64_t bg = __ballot(x > prefix), be = __ballot(x == prefix), below = (1ull << lane) - 1;
        const unsigned g = gt + __popcll(bg & below), e = eq + __popcll(be & below);
        if (x > prefix || (x == prefix && e < left)) out[g + min(e, left)] = j0 + 64 * r;
        gt += __popcll(bg);
        eq += __popcll(be);
    };
#pragma unroll
    for (int r = 0; r < kRowsRegs; ++r) {
        if (r < rounds) place(k[r], r);
    }
    for (int r = kRowsRegs; r < rounds; ++r) place(key_at(r), r);
}

// ---------------------------------------------------------------------------
// Compaction.  A workgroup takes 16 kept rows of one (sequence, kv head), the
// rows of one destination page.
template <typename T>
__device__ __forceinline__ void compact_body(const CompactArgs& a) {
    __shared__ int64_t s_src[kPageRows];  // source page of the pool * 16 + row in it, -1: no row
    __shared__ int s_to;
    const int tid = threadIdx.x, kv = a.n_kv_head;
    const int64_t unit = blockIdx.x, sk = unit / a.n_grid;
    const int jp = (int)(unit - sk * a.n_grid), s = (int)(sk / kv), h = (int)(sk - (int64_t)s * kv);
    const int len = max(a.lengths[s], 0);
    if (tid < kPageRows) {
        const int j = jp * kPageRows + tid;
        const int row = j < a.keep ? a.kept[sk * a.keep + j] : -1;
        int64_t src = -1;
        if (row >= 0 && row < len && row < (int64_t)a.max_pages * kPageRows) {
            const int page = a.block_table[(size_t)s * a.max_pages + (row >> kPageShift)];
            if (page < 0 || page >= a.n_pages) atomicOr(a.err, 4);
            src = (int64_t)min(max(page, 0), a.n_pages - 1) * kPageRows + (row & (kPageRows - 1));
        } else if (row != -1) {
            atomicOr(a.err, 4);
        }
        const uint64_t any = __ballot(src >= 0);
        if (tid == 0) {
            int to = -1;
            if (any) {
                to = a.to_table[(size_t)s * a.to_pages + jp];
                if (to < 0 || to >= a.n_pages) {
                    atomicOr(a.err, 4);
                    to = -1;
                }
            }
            s_to = to;
        }
        s_src[tid] = src;
        if (a.weights_out && j < a.keep)
            a.weights_out[sk * a.weight_stride + j] = src >= 0 ? a.weights_in[sk * a.weight_stride + row] : 0.f;
    }
    __syncthreads();
    if (a.weights_out && jp == a.n_grid - 1)  // what follows the last kept row
        for (int64_t j = a.keep + tid; j < a.weight_stride; j += 256) a.weights_out[sk * a.weight_stride + j] = 0.f;
    const int to = s_to;
    if (to < 0) return;
    const size_t page_bytes = PageFmt<T>::page(kv), head = PageFmt<T>::head(h), row_bytes = PageFmt<T>::row(kv);
    if constexpr (__is_same(T, q4_t)) {
        for (int i = tid; i < 2 * 16 * 8; i += 256) {  // a slot of 8 lanes moves a row
            const int v = i >> 7, r = i >> 3 & 15, c = i & 7;
            const int64_t src = s_src[r];
            if (src < 0) continue;
            char* pool = v ? a.v_pages : a.k_pages;
            const char* from = pool + (src >> kPageShift) * page_bytes + head;
            char* dst = pool + (size_t)to * page_bytes + head;
            const int r1 = (int)src & (kPageRows - 1);
            if (v) {
                const int p0 = (r & 3) == 1 ? 2 : (r & 3) == 2 ? 1 : r & 3, p1 = (r1 & 3) == 1 ? 2 : (r1 & 3) == 2 ? 1 : r1 & 3;
                for (int k = c; k < 32; k += 8)  // byte k of the row
                    dst[8 * (16 * (r >> 2) + (k & 15)) + 4 * (k >> 4) + p0] =
                        from[8 * (16 * (r1 >> 2) + (k & 15)) + 4 * (k >> 4) + p1];
                if (c < 2)
                    reinterpret_cast<uint16_t*>(dst)[256 + 8 * (r >> 2) + 4 * c + (r & 3)] =
                        reinterpret_cast<const uint16_t*>(from)[256 + 8 * (r1 >> 2) + 4 * c + (r1 & 3)];
            } else {
                const int g = c >> 1, m = c & 1;
                *reinterpret_cast<unsigned*>(dst + 8 * (16 * g + r) + 4 * m) =
                    *reinterpret_cast<const unsigned*>(from + 8 * (16 * g + r1) + 4 * m);
                if (c < 2)
                    reinterpret_cast<uint16_t*>(dst)[256 + 16 * c + r] =
                        reinterpret_cast<const uint16_t*>(from)[256 + 16 * c + r1];
            }
        }
    } else {
        constexpr int HB = CacheFmt<T>::kHeadBytes, CH = HB % 16 ? 4 : 16, PER = HB / CH;
        using Word = std::conditional_t<CH == 16, u32x4, unsigned>;
        for (int i = tid; i < 2 * kPageRows * PER; i += 256) {
            const int v = i / (kPageRows * PER), k = i - v * kPageRows * PER, r = k / PER, c = k - r * PER;
            const int64_t src = s_src[r];
            if (src < 0) continue;
            char* pool = v ? a.v_pages : a.k_pages;
            *reinterpret_cast<Word*>(pool + (size_t)to * page_bytes + r * row_bytes + head + c * CH) =
                *reinterpret_cast<const Word*>(pool + (src >> kPageShift) * page_bytes +
                                               (src & (kPageRows - 1)) * row_bytes + head + c * CH);
        }
    }
}
