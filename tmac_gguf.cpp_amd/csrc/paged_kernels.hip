// paged_kernels.hip -- gfx950 kernels of the serving operators on 16-row paged
// caches: appending rotated rows, per-page key bounds, page selection, and
// decode attention over selected pages or over shared prefixes.
//
// All take head_dim 64, any number of kv heads and up to kMaxGroupHeads query
// heads per kv head at run time; a kernel is built per cache element type.
#include <hip/hip_runtime.h>

#include "attn_args.h"
#include "attn_device.h"

using namespace tmac;

namespace {

// ---------------------------------------------------------------------------
// Append.  A workgroup takes rows_per_group consecutive rows.  Every thread
// looks at its share of row_starts once: an entry at or before the first row
// raises the sequence of that row, an entry inside raises that row's, so a
// running maximum over the rows gives each its sequence (the last one that
// starts at or before it; empty sequences never win).  The rows' positions and
// pages go to LDS, then slots of 8 lanes (8 dims a lane) take the rows' heads:
// n_head query heads (rotated to q_out), n_kv_head keys (rotated, to the
// cache) and n_kv_head values.  Rotation and storage are the layer step's
// (rope8, put_row), so a row's bytes do not depend on which call wrote it.
template <typename T>
__device__ __forceinline__ void append_body(const AppendArgs& a) {
    __shared__ int s_seq[kAppendRows];
    __shared__ int s_pos[kAppendRows];
    __shared__ int64_t s_row[kAppendRows];  // pool row, -1: not stored
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
        int pos = -1;
        int64_t row = -1;
        if (s >= 0 && s < a.n_seq) {  // entry n_seq: rows behind the last sequence
            const int64_t p = (int64_t)a.positions[s] + (t0 + tid - a.row_starts[s]);
            if (p >= 0 && p < a.capacity) {
                pos = (int)p;
                const int page = a.block_table[(size_t)s * a.max_pages + (pos >> kPageShift)];
                if (page >= 0 && page < a.n_pages)
                    row = (int64_t)page * kPageRows + (pos & (kPageRows - 1));
                else
                    atomicOr(a.err, 4);
            } else {
                atomicOr(a.err, 1);
            }
        }
        s_pos[tid] = pos;
        s_row[tid] = row;
    }
    __syncthreads();
    const int c = tid & 7, slot = tid >> 3;
    const int nh = a.q ? a.n_head : 0, kv = a.n_kv_head, per = nh + 2 * kv;
    constexpr int HB = CacheFmt<T>::kHeadBytes, DB = CacheFmt<T>::kDimBytes;
    for (int it = slot; it < n * per; it += 32) {
        const int r = it / per, h = it - r * per, pos = s_pos[r];
        if (pos < 0) continue;
        const int64_t t = t0 + r, row = s_row[r];
        float x[8];
        if (h < nh) {
            load8(x, a.q + t * a.q_stride + h * kHeadDim + 4 * c);
            rope8(x, a.rope_cs + (size_t)pos * (kHeadDim / 2), c);
            store8(a.q_out + (t * nh + h) * kHeadDim + 4 * c, x);
        } else if (row >= 0) {
            const bool key = h < nh + kv;
            const int hk = key ? h - nh : h - nh - kv;
            load8(x, (key ? a.k + t * a.k_stride : a.v + t * a.v_stride) + hk * kHeadDim + 4 * c);
            if (key) rope8(x, a.rope_cs + (size_t)pos * (kHeadDim / 2), c);
            char* p = (key ? a.k_pages : a.v_pages) + (row * kv + hk) * HB + 4 * c * DB;
            put_row<T>(x, p, c, true);
        }
    }
}

// ---------------------------------------------------------------------------
// Page bounds.  One wave per (sequence, page, kv head): a slot of 8 lanes reads
// a row, 8 dims a lane, rows slot and slot + 8; the running max and min go
// over the slots with three lane exchanges.
//
// bf16 rounded outward: the fp32 value with its low half cut is the bf16 next
// to it toward zero, and adding one to the cut word steps away from zero.  A
// value beyond the largest finite bf16 becomes that, a NaN makes the dim's
// bounds the whole range: bounds are always finite.
__device__ __forceinline__ unsigned bf16_above(float x, bool up) {
    const unsigned u = __float_as_uint(x);
    const bool neg = u >> 31;
    unsigned t = (u & 0x7FFFFFFFu) >> 16;
    if ((u & 0xFFFFu) && neg != up) t++;
    return min(t, 0x7F7Fu) | (neg ? 0x8000u : 0u);
}

template <typename T>
__device__ __forceinline__ void bounds_body(const BoundsArgs& a) {
    const int lane = threadIdx.x & 63, c = lane & 7, slot = lane >> 3;
    const int64_t item = (int64_t)blockIdx.x * kPagedWaves + (threadIdx.x >> 6);
    const int kv = a.n_kv_head;
    const int64_t per_seq = (int64_t)a.n_grid * kv;
    if (item >= per_seq * a.n_seq) return;
    const int s = (int)(item / per_seq), rest = (int)(item - s * per_seq), i = rest / kv, h = rest - i * kv;
    const int len = a.lengths[s], first = a.first_rows ? max(a.first_rows[s], 0) : 0;
    if (first >= len) return;
    if (len - first > a.max_new || len > (int64_t)a.max_pages * kPageRows) {
        if (rest == 0 && lane == 0) atomicOr(a.err, 2);
        return;
    }
    const int j = (first >> kPageShift) + i;
    const int n = min(kPageRows, len - j * kPageRows);
    if (n <= 0) return;
    const int page = a.block_table[(size_t)s * a.max_pages + j];
    if (page < 0 || page >= a.n_pages) {
        if (lane == 0) atomicOr(a.err, 4);
        return;
    }
    constexpr int HB = CacheFmt<T>::kHeadBytes, DB = CacheFmt<T>::kDimBytes;
    const char* base = a.k_pages + ((size_t)page * kPageRows * kv + h) * HB + 4 * c * DB;
    float hi[8], lo[8];
    unsigned bad = 0;
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        hi[t] = kNegInf;
        lo[t] = -kNegInf;
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int r = slot + 8 * u;
        float x[8];
        load_row<T, false>(x, base + (size_t)min(r, n - 1) * kv * HB, c);  // a row beyond the last repeats it
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            hi[t] = fmaxf(hi[t], x[t]);
            lo[t] = fminf(lo[t], x[t]);
            bad |= (x[t] == x[t] ? 0u : 1u) << t;
        }
    }
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        hi[t] = xor_max<8>(hi[t]);
        lo[t] = -xor_max<8>(-lo[t]);
    }
    bad |= __shfl_xor(bad, 8);
    bad |= __shfl_xor(bad, 16);
    bad |= __shfl_xor(bad, 32);
    if (slot < 2) {  // slot 0 writes the largest values, slot 1 the smallest
        uint16_t b[8];
#pragma unroll
        for (int t = 0; t < 8; ++t)
            b[t] = (uint16_t)((bad >> t & 1) ? (slot ? 0xFF7Fu : 0x7F7Fu) : bf16_above(slot ? lo[t] : hi[t], slot == 0));
        uint16_t* o = a.bounds + ((size_t)page * kv + h) * (kBoundsBytes / 2) + slot * kHeadDim + 4 * c;
#pragma unroll
        for (int t = 0; t < 2; ++t)
            *reinterpret_cast<u32x2*>(o + 32 * t) = u32x2{(unsigned)b[4 * t] | (unsigned)b[4 * t + 1] << 16,
                                                         (unsigned)b[4 * t + 2] | (unsigned)b[4 * t + 3] << 16};
    }
}

// ---------------------------------------------------------------------------
// Page selection.  A page's score for a kv head is the largest, over the
// group's query heads, of sum_d max(q_d hi_d, q_d lo_d): no key of the page
// has a larger q . k.  The sum runs in 64 bits and is rounded once, so scores,
// and with them the selection, do not depend on the order of the sum (up to
// 2^-53).  max(q hi, q lo) is q times hi where q >= 0 and times lo elsewhere; a
// bf16 value as a double has a low word of zero, so one bit select of the high
// words picks the factor.
//
// Slot of 8 lanes = one page, 8 dims a lane; the queries' 8 dims of every head
// stay in registers over the workgroup's kScorePages pages.
__device__ __forceinline__ double slot_sum64(double x) {
#pragma unroll
    for (int m = 1; m < 8; m *= 2) x += __shfl_xor(x, m);
    return x;
}

// fp32 -> unsigned of the same order; NaN as +infinity.
__device__ __forceinline__ unsigned order_key(float x) {
    const unsigned u = x == x ? __float_as_uint(x) : 0x7F800000u;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int select_pages_of(const SelectArgs& a, int s) {  // -1: a bad length
    const int len = max(a.lengths[s], 0);
    return len > a.max_len ? -1 : (len + kPageRows - 1) >> kPageShift;
}

template <int GT>
__device__ __forceinline__ void score_body(const SelectArgs& a) {
    const int lane = threadIdx.x & 63, c = lane & 7, slot = threadIdx.x >> 3;
    const int kv = a.n_kv_head, G = a.n_head / kv;
    const int chunk = blockIdx.x % a.chunks, sk = blockIdx.x / a.chunks, s = sk / kv, h = sk - s * kv;
    const int n = select_pages_of(a, s);
    const int j0 = chunk * kScorePages, j1 = min(n, j0 + kScorePages);
    if (n <= a.top || j0 >= j1) return;  // every page is taken, or none left
    for (int g0 = 0; g0 < G; g0 += GT) {
        double q[GT][8];
        unsigned up[GT][8];  // all ones where the query value is not negative
#pragma unroll
        for (int g = 0; g < GT; ++g) {
            float x[8];
            const float* p = a.q + ((size_t)s * a.n_head + h * G + min(g0 + g, G - 1)) * kHeadDim + 8 * c;
            const float4 u = *reinterpret_cast<const float4*>(p), w = *reinterpret_cast<const float4*>(p + 4);
            x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
            x[4] = w.x; x[5] = w.y; x[6] = w.z; x[7] = w.w;
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                q[g][t] = (double)x[t];
                up[g][t] = x[t] < 0.f ? 0u : ~0u;
            }
        }
        for (int j = j0 + slot; j < j1; j += 32) {
            int page = a.block_table[(size_t)s * a.max_pages + j];
            if (page < 0 || page >= a.n_pages) {
                if (c == 0) atomicOr(a.err, 4);
                page = min(max(page, 0), a.n_pages - 1);
            }
            const uint16_t* b = a.bounds + ((size_t)page * kv + h) * (kBoundsBytes / 2) + 8 * c;
            const u32x4 uh = *reinterpret_cast<const u32x4*>(b), ul = *reinterpret_cast<const u32x4*>(b + kHeadDim);
            double sum[GT];
#pragma unroll
            for (int g = 0; g < GT; ++g) sum[g] = 0.0;
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const unsigned hi = __double2hiint(__uint_as_float(t & 1 ? uh[t / 2] & 0xFFFF0000u : uh[t / 2] << 16));
                const unsigned lo = __double2hiint(__uint_as_float(t & 1 ? ul[t / 2] & 0xFFFF0000u : ul[t / 2] << 16));
#pragma unroll
                for (int g = 0; g < GT; ++g) {
                    const unsigned x = (hi & up[g][t]) | (lo & ~up[g][t]);
                    sum[g] = __builtin_fma(q[g][t], __hiloint2double((int)x, 0), sum[g]);
                }
            }
            unsigned best = 0;
#pragma unroll
            for (int g = 0; g < GT; ++g) best = max(best, order_key((float)slot_sum64(sum[g])));
            if (c == 0) {
                unsigned* key = a.keys + (size_t)sk * a.key_stride + j;
                *key = g0 ? max(*key, best) : best;
            }
        }
    }
}

// The top pages of one (sequence, kv head), ascending.  Digit by digit from the
// top, a histogram of the keys that agree with the digits found so far gives
// the digit of the top-th largest key; then one pass in page order takes the
// keys above it and the first of those equal to it.
constexpr int kSelectThreads = 256;
__device__ __forceinline__ unsigned key_of(const SelectArgs& a, const unsigned* keys, int j, int n) {
    return j < a.first || j >= n - a.last ? 0xFFFFFFFFu : keys[j];
}

__device__ __forceinline__ void select_body(const SelectArgs& a) {
    __shared__ unsigned s_hist[256];
    __shared__ unsigned s_prefix, s_left;
    __shared__ int s_gt[kSelectThreads / 64], s_eq[kSelectThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int sk = blockIdx.x, s = sk / a.n_kv_head;
    const int n = select_pages_of(a, s);
    int32_t* out = a.selected + (size_t)sk * a.top;
    if (n < 0 && tid == 0) atomicOr(a.err, 2);
    if (n <= a.top) {
        for (int i = tid; i < a.top; i += kSelectThreads) out[i] = i < n ? i : -1;
        return;
    }
    const unsigned* keys = a.keys + (size_t)sk * a.key_stride;
    unsigned prefix = 0, left = (unsigned)a.top;  // keys still to take among those that agree with prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
        s_hist[tid] = 0;
        __syncthreads();
        for (int j = tid; j < n; j += kSelectThreads) {
            const unsigned k = key_of(a, keys, j, n);
            if (shift == 24 || k >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&s_hist[k >> shift & 255], 1u);
        }
        __syncthreads();
        if (tid < 64) {  // lane l: digits 255 - 4 l .. 252 - 4 l, from the top
            unsigned cnt[4], sum = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += cnt[i] = s_hist[255 - 4 * lane - i];
            unsigned incl = sum;
#pragma unroll
            for (int m = 1; m < 64; m *= 2) {
                const unsigned o = __shfl_up(incl, m);
                if (lane >= m) incl += o;
            }
            unsigned above = incl - sum;
            if (above < left && incl >= left) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (above < left && above + cnt[i] >= left) {
                        s_prefix = prefix | (unsigned)(255 - 4 * lane - i) << shift;
                        s_left = left - above;
                    }
                    above += cnt[i];
                }
            }
        }
        __syncthreads();
        prefix = s_prefix;
        left = s_left;
    }
    int n_gt = 0, n_eq = 0;  // taken so far, equal keys seen so far
    for (int j0 = 0; j0 < n; j0 += kSelectThreads) {
        const int j = j0 + tid;
        const unsigned k = j < n ? key_of(a, keys, j, n) : 0;
        const bool gt = j < n && k > prefix, eq = j < n && k == prefix;
        const uint64_t bg = __ballot(gt), be = __ballot(eq), below = (1ull << lane) - 1;
        __syncthreads();
        if (lane == 0) {
            s_gt[wave] = __popcll(bg);
            s_eq[wave] = __popcll(be);
        }
        __syncthreads();
        int g = n_gt, e = n_eq;  // before this thread's page
        for (int w = 0; w < kSelectThreads / 64; ++w) {
            if (w < wave) g += s_gt[w], e += s_eq[w];
            n_gt += s_gt[w], n_eq += s_eq[w];
        }
        g += __popcll(bg & below);
        e += __popcll(be & below);
        if (gt || (eq && e < (int)left)) out[g + min(e, (int)left)] = j;
    }
}

// ---------------------------------------------------------------------------
// Decode attention by (columns, kv head, run of pages) on fp32 MFMA
// (v_mfma_f32_16x16x4_f32, products and sums of fp32: the cache rows are
// widened exactly, so every cache type gets the fp32 result).  A tile is one
// page, 16 keys x 16 columns; a column is a query head of one sequence.
//   S^T (16 keys x 16 columns) = K (keys x dims) . Q^T.   Lane (i = l % 16,
//     g = l / 16) holds key i's dims 32 m + 8 g + e of K and column i's of Q:
//     step (m, e) contracts the four dims 32 m + 8 g + e, g = 0..3.
//   P^T = exp2(S^T - m), online per column with a lazy maximum.
//   O^T (64 dims x 16 columns) += V^T . P^T.  The accumulator S^T leaves keys
//     4 g + r, r = 0..3, in lane group g, so step r contracts the keys 4 g + r
//     straight from the same registers; row i of block b is dim 4 i + b, so
//     lane (i, g) reads V of key 4 g + r as the four dims 4 i + 0..3.
// No operand passes through LDS or another lane.
template <typename T>
struct Tile {};
template <>
struct Tile<float> {
    f32x4 k[4], v[4];
};
template <>
struct Tile<__bf16> {
    u32x4 k[2];
    u32x2 v[4];
};
template <>
struct Tile<_Float16> {
    u32x4 k[2];
    u32x2 v[4];
};
template <>
struct Tile<q8_0_t> {
    unsigned k[4], kd, v[4], vd[4];
};

// kp / vp: row 0 of the page's head; stride: bytes between rows.
template <typename T>
__device__ __forceinline__ void tile_load(Tile<T>& t, const char* kp, const char* vp, int stride, int lane) {
    const int i = lane & 15, g = lane >> 4;
    const char* kr = kp + i * stride;
    constexpr int DB = CacheFmt<T>::kDimBytes;
    if constexpr (__is_same(T, float)) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            t.k[2 * m] = *reinterpret_cast<const f32x4*>(kr + (32 * m + 8 * g) * DB);
            t.k[2 * m + 1] = *reinterpret_cast<const f32x4*>(kr + (32 * m + 8 * g + 4) * DB);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) t.v[r] = *reinterpret_cast<const f32x4*>(vp + (4 * g + r) * stride + 4 * i * DB);
    } else if constexpr (__is_same(T, q8_0_t)) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            t.k[2 * m] = *reinterpret_cast<const unsigned*>(kr + 32 * m + 8 * g);
            t.k[2 * m + 1] = *reinterpret_cast<const unsigned*>(kr + 32 * m + 8 * g + 4);
        }
        t.kd = *reinterpret_cast<const unsigned*>(kr + 64);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            t.v[r] = *reinterpret_cast<const unsigned*>(vp + (4 * g + r) * stride + 4 * i);
            t.vd[r] = *reinterpret_cast<const unsigned*>(vp + (4 * g + r) * stride + 64);
        }
    } else {
#pragma unroll
        for (int m = 0; m < 2; ++m) t.k[m] = *reinterpret_cast<const u32x4*>(kr + (32 * m + 8 * g) * DB);
#pragma unroll
        for (int r = 0; r < 4; ++r) t.v[r] = *reinterpret_cast<const u32x2*>(vp + (4 * g + r) * stride + 4 * i * DB);
    }
}

template <typename T>
__device__ __forceinline__ float half16(unsigned w, int e) {  // element e (0, 1) of a word of 16-bit values
    if constexpr (__is_same(T, __bf16))
        return __uint_as_float(e ? w & 0xFFFF0000u : w << 16);
    else
        return half_bits_to_float(e ? w >> 16 : w & 0xFFFFu);
}

// Element (m, e) of the K operand; element b of the V operand of step r.
template <typename T>
__device__ __forceinline__ float tile_k(const Tile<T>& t, int m, int e) {
    if constexpr (__is_same(T, float))
        return t.k[2 * m + e / 4][e % 4];
    else if constexpr (__is_same(T, q8_0_t))
        return (float)(signed char)(t.k[2 * m + e / 4] >> (8 * (e % 4))) *
               half_bits_to_float(m ? t.kd >> 16 : t.kd & 0xFFFFu);
    else
        return half16<T>(t.k[m][e / 2], e % 2);
}
template <typename T>
__device__ __forceinline__ float tile_v(const Tile<T>& t, int r, int b, int i) {
    if constexpr (__is_same(T, float))
        return t.v[r][b];
    else if constexpr (__is_same(T, q8_0_t))
        return (float)(signed char)(t.v[r] >> (8 * b)) * half_bits_to_float(i < 8 ? t.vd[r] & 0xFFFFu : t.vd[r] >> 16);
    else
        return half16<T>(t.v[r][b / 2], b % 2);
}

constexpr float kNoMax = -__FLT_MAX__;  // running maximum of a column that has met no key

// One wave's state of a block of 16 columns.
struct Cols {
    float q[16];
    f32x4 o[4];   // block b, row r: dim 16 g + 4 r + b
    float m, l;   // m: the column's (equal in the four lane groups); l: this lane's keys
};

// One tile: keys lo .. hi - 1 of the page take part.
template <typename T>
__device__ __forceinline__ void attend_tile(Cols& st, const Tile<T>& t, int lo, int hi, int lane) {
    const int i = lane & 15, g = lane >> 4;
    const bool full = lo <= 0 && hi >= kPageRows;
    f32x4 s = {0.f, 0.f, 0.f, 0.f}, s1 = s;  // two sums: a chain of 16 dependent products would wait on itself
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        s = __builtin_amdgcn_mfma_f32_16x16x4f32(tile_k<T>(t, 0, e), st.q[e], s, 0, 0, 0);
        s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(tile_k<T>(t, 1, e), st.q[8 + e], s1, 0, 0, 0);
    }
    s += s1;
    if (!full) {
#pragma unroll
        for (int r = 0; r < 4; ++r) s[r] = 4 * g + r >= lo && 4 * g + r < hi ? s[r] : kNegInf;
    }
    const float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
    if (__any(top > st.m + kTau || st.m == kNoMax)) {
        const float m1 = fmaxf(st.m, max4_rows(top));
        const float w = fast_exp2(st.m - m1);
        st.m = m1;
        st.l *= w;
#pragma unroll
        for (int b = 0; b < 4; ++b) st.o[b] *= w;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) s[r] = fast_exp2(s[r] - st.m);
    st.l += (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const bool in = full || (4 * g + r >= lo && 4 * g + r < hi);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const float vx = in ? tile_v<T>(t, r, b, i) : 0.f;  // a row outside may hold anything
            st.o[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(vx, s[r], st.o[b], 0, 0, 0);
        }
    }
}

// A run of tiles.  look(e, logical, page) gives entry e (0 <= e < n) its page of
// the pool (checked, in range) and its logical page index (-1: skipped); rows
// row_lo .. row_hi - 1 of the sequence take part.  The NW waves take the
// entries in turn; a wave looks up 64 of its entries at a time, one a lane.
template <typename T, int NW, typename Look>
__device__ __forceinline__ void attend_run(Cols& st, const PagedAttnArgs& a, int h, int n, int64_t row_lo,
                                           int64_t row_hi, int wave, int lane, Look look) {
    constexpr int HB = CacheFmt<T>::kHeadBytes;
    const int stride = a.n_kv_head * HB;
    const size_t page_bytes = (size_t)kPageRows * stride;
    const int mine = (n - wave + NW - 1) / NW;  // this wave's entries
    for (int c0 = 0; c0 < mine; c0 += 64) {
        const int cnt = min(64, mine - c0);
        int logical = -1, page = 0;
        if (lane < cnt) look((c0 + lane) * NW + wave, logical, page);
        Tile<T> t[2];
        auto fetch = [&](Tile<T>& x, int e) {
            const size_t at = (size_t)__builtin_amdgcn_readlane(page, e) * page_bytes + (size_t)h * HB;
            tile_load<T>(x, a.k_pages + at, a.v_pages + at, stride, lane);
        };
        fetch(t[0], 0);
        for (int e = 0; e < cnt; e += 2) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if (e + u < cnt) {
                    fetch(t[1 - u], min(e + u + 1, cnt - 1));
                    const int j = __builtin_amdgcn_readlane(logical, e + u);
                    const int64_t r0 = (int64_t)j * kPageRows;
                    const int lo = (int)max((int64_t)0, min(row_lo - r0, (int64_t)kPageRows));
                    const int hi = j < 0 ? 0 : (int)max((int64_t)0, min(row_hi - r0, (int64_t)kPageRows));
                    if (hi > lo) attend_tile<T>(st, t[u], lo, hi, lane);
                }
            }
        }
    }
}

// Empty columns with the query rows p (null: an unused column), scaled.
__device__ __forceinline__ void cols_init(Cols& st, const float* p, float scale, int lane) {
    const int g = lane >> 4;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
        if (p) {
            x = *reinterpret_cast<const float4*>(p + 32 * m + 8 * g);
            y = *reinterpret_cast<const float4*>(p + 32 * m + 8 * g + 4);
        }
        float* o = st.q + 8 * m;
        o[0] = x.x * scale; o[1] = x.y * scale; o[2] = x.z * scale; o[3] = x.w * scale;
        o[4] = y.x * scale; o[5] = y.y * scale; o[6] = y.z * scale; o[7] = y.w * scale;
    }
    st.m = kNoMax;
    st.l = 0.f;
#pragma unroll
    for (int b = 0; b < 4; ++b) st.o[b] = f32x4{0.f, 0.f, 0.f, 0.f};
}

// Merges the NW waves through LDS and hands every column's maximum, sum and
// four dims to put(column, first dim, m, l, acc): one call a thread of the first
// 256 (16 columns x 16 dim quads).
template <int NW>
struct MergeLds {
    alignas(16) float o[NW][16][kHeadDim + 4];
    float m[NW][16], l[NW][16];
};
template <int NW, typename Put>
__device__ __forceinline__ void merge_waves(Cols& st, MergeLds<NW>& lds, int wave, int lane, Put put) {
    const int i = lane & 15, g = lane >> 4;
    const float l = sum4_rows(st.l);
    if (g == 0) {
        lds.m[wave][i] = st.m;
        lds.l[wave][i] = l;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
        *reinterpret_cast<f32x4*>(&lds.o[wave][i][16 * g + 4 * r]) =
            f32x4{st.o[0][r], st.o[1][r], st.o[2][r], st.o[3][r]};
    __syncthreads();
    const int c = threadIdx.x >> 4, d = 4 * (threadIdx.x & 15);
    if (c >= 16) return;
    float M = lds.m[0][c];
#pragma unroll
    for (int w = 1; w < NW; ++w) M = fmaxf(M, lds.m[w][c]);
    float L = 0.f;
    f32x4 A = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        const float x = fast_exp2(lds.m[w][c] - M);
        L += x * lds.l[w][c];
        A += x * *reinterpret_cast<const f32x4*>(&lds.o[w][c][d]);
    }
    put(c, d, M, L, A);
}

__device__ __forceinline__ f32x4 finish_row(f32x4 acc, float l) {
    return l == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : acc / l;
}

// Partials: every row's slots of 64 sums, then every row's slots of (m, l).
__device__ __forceinline__ void put_partial(const PagedAttnArgs& a, int64_t row, int slot, int d, float M, float L,
                                            f32x4 A) {
    const size_t at = (size_t)row * a.n_slots + slot;
    *reinterpret_cast<f32x4*>(a.ws + at * kHeadDim + d) = A;
    if (d == 0)
        *reinterpret_cast<float2*>(a.ws + (size_t)a.n_seq * a.n_head * a.n_slots * kHeadDim + 2 * at) =
            make_float2(M, L);
}

// Over a list: workgroup (split, kv head, sequence).
template <typename T>
__device__ __forceinline__ void selected_body(const PagedAttnArgs& a) {
    constexpr int NW = kPagedWaves;
    __shared__ MergeLds<NW> lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kv = a.n_kv_head, G = a.group;
    const int split = blockIdx.x % a.n_slots, sk = blockIdx.x / a.n_slots, s = sk / kv, h = sk - s * kv;
    const int len = a.lengths[s];
    const int e0 = split * a.per_split, n = min(a.per_split, a.top - e0);
    const int32_t* list = a.selected + (size_t)sk * a.top + e0;
    const int32_t* table = a.block_table + (size_t)s * a.max_pages;
    const int64_t row0 = (int64_t)s * a.n_head + h * G;
    const int col = lane & 15;
    Cols st;
    cols_init(st, col < G ? a.q + (row0 + col) * kHeadDim : nullptr, a.qscale, lane);
    attend_run<T, NW>(st, a, h, n, 0, len, wave, lane, [&](int e, int& logical, int& page) {
        const int j = list[e];
        if (j == -1) return;
        if (j < 0 || j >= a.max_pages) {
            atomicOr(a.err, 4);
            return;
        }
        if ((int64_t)j * kPageRows >= len) return;  // behind the last row
        page = table[j];
        if (page < 0 || page >= a.n_pages) {
            atomicOr(a.err, 4);
            page = min(max(page, 0), a.n_pages - 1);
        }
        logical = j;
    });
    merge_waves<NW>(st, lds, wave, lane, [&](int c, int d, float M, float L, f32x4 A) {
        if (c >= G) return;
        if (a.n_slots == 1)
            *reinterpret_cast<f32x4*>(a.out + (row0 + c) * kHeadDim + d) = finish_row(A, L);
        else
            put_partial(a, row0 + c, split, d, M, L, A);
    });
}

// Merge of one row's partials, slots 0 .. n0 - 1 and skip_to .. skip_to + n1 - 1,
// by WPR waves: a wave reads four slots at once, 16 lanes of four dims each, 64
// slots (WPR = 4) or 16 (WPR = 1) in one round of independent loads.  The
// result is in the lanes 0 .. 15 of the row's first wave.  Every thread calls it.
template <int WPR>
__device__ __forceinline__ f32x4 merge_slots(const PagedAttnArgs& a, int64_t row, int n0, int skip_to, int n1, int w,
                                             int lane, float& L) {
    constexpr int kRound = 16 * WPR;
    const int n = n0 + n1, sub = lane >> 4;
    const float* acc = a.ws + (size_t)row * a.n_slots * kHeadDim + 4 * (lane & 15);
    const float2* ml = reinterpret_cast<const float2*>(a.ws + (size_t)a.n_seq * a.n_head * a.n_slots * kHeadDim) +
                       (size_t)row * a.n_slots;
    auto slot = [&](int e) { return e < n0 ? e : skip_to + e - n0; };
    float M = kNoMax;
    f32x4 A = {0.f, 0.f, 0.f, 0.f};
    L = 0.f;
    for (int c0 = 0; c0 < n; c0 += kRound) {
        f32x4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = c0 + 4 * (WPR * i + w) + sub;
            v[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (e < n) v[i] = *reinterpret_cast<const f32x4*>(acc + (size_t)slot(e) * kHeadDim);
        }
        float2 x = make_float2(kNoMax, 0.f);
        if (lane < kRound && c0 + lane < n) x = ml[slot(c0 + lane)];
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
    return A;
}

template <int WPR>
__device__ __forceinline__ void selected_merge_body(const PagedAttnArgs& a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = (int64_t)blockIdx.x * (kPagedWaves / WPR) + wave / WPR;
    if (row >= (int64_t)a.n_seq * a.n_head) return;
    float L;
    const f32x4 A = merge_slots<WPR>(a, row, a.n_slots, a.n_slots, 0, wave % WPR, lane, L);
    if (wave % WPR == 0 && lane < 16) *reinterpret_cast<f32x4*>(a.out + row * kHeadDim + 4 * lane) = finish_row(A, L);
}

// A lane's group: its sequences [first, end), clamped into the batch, and its
// prefix.  All of a group's numbers are loaded together: in these short kernels
// every dependent load is a good part of a microsecond.
struct Group {
    int first, end, prefix;
};
__device__ __forceinline__ Group group_at(const PagedAttnArgs& a, int g) {
    Group r = {0, 0, 0};
    if (g < a.n_groups) {
        const int s0 = a.group_starts[g], s1 = a.group_starts[g + 1];
        r.prefix = max(a.prefix_lens[g], 0);
        r.first = min(max(s0, 0), a.n_seq);
        r.end = min(max(s1, r.first), a.n_seq);
    }
    return r;
}

// A sequence's rows: [0, prefix) through its group's first sequence, [prefix,
// len) through its own pages.  Its group is the last one that holds it.
struct SharedSeq {
    int64_t prefix, len;
    bool bad;  // a length or prefix outside what the launch covers
};
__device__ __forceinline__ SharedSeq shared_seq(const PagedAttnArgs& a, int s, int lane) {
    SharedSeq r;
    r.len = max(a.lengths[s], 0);
    r.prefix = 0;
    for (int g0 = 0; g0 < a.n_groups; g0 += 64) {
        const Group g = group_at(a, g0 + lane);
        const uint64_t b = __ballot(s >= g.first && s < g.end);
        if (b) r.prefix = __builtin_amdgcn_readlane(g.prefix, 63 - __clzll(b));
    }
    r.bad = r.len > 0 && (r.prefix > a.max_prefix || r.len < r.prefix || r.len - r.prefix > a.max_tail ||
                          r.len > (int64_t)a.max_pages * kPageRows);
    return r;
}

// Pages of one run of a prefix of `prefix` rows cut into prefix_splits runs.
__device__ __forceinline__ int prefix_run_pages(const PagedAttnArgs& a, int64_t prefix) {
    const int n = (int)((prefix + kPageRows - 1) >> kPageShift), runs = max(1, a.prefix_splits);
    return max(1, (n + runs - 1) / runs);
}

// ---------------------------------------------------------------------------
// Shared prefix on 16-bit MFMA (v_mfma_f32_16x16x32).  A workgroup of 8 waves
// takes 64 columns, (sequence, query head) pairs of one group and kv head, over
// a run of the prefix: wave (kg, cw) the columns 32 cw .. 32 cw + 31 and, of
// every stage, the keys of quarter kg.  What bounds it is the products: every fp32
// operand is carried by 16-bit parts that together hold its 24 bits, so fp32
// accuracy costs a multiple of the plain product,
//   cache   K, V        q            P            products, Q.K and P.V
//   bf16    exact       3 bf16       3 bf16       3, 3
//   fp16    exact       2 fp16       2 fp16       2, 2
//   Q8_0    int8 exact  2 fp16       3 bf16 x 2   2, 3 (scales on S and on P)
//   fp32    3 bf16      3 bf16       3 bf16       6, 6 (parts i + j <= 2; the rest is below 2^-24)
// against fp32 MFMA at 1/16 of the 16-bit rate.  (Two bf16 parts of P, 2^-18,
// left 2e-6 of the output's norm.)
//
// A stage's K and V rows go through registers (fetched one stage ahead) to LDS
// once, converted there, and feed both column waves; V is read back transposed
// (ds_read_b64_tr_b16).  16-byte chunks of a 128-byte LDS row are XORed with
// the row, K by row & 7, V by 2 row & 7, so that both reads touch all banks.
template <typename T>
struct Px;
template <>
struct Px<__bf16> {
    using KOps = MMath<__bf16>;
    using VOps = MMath<__bf16>;
    static constexpr int kParts = 1, kQ = 3, kP = 3, kSets = 1, kKeys = 64;
};
template <>
struct Px<_Float16> {
    using KOps = MMath<_Float16>;
    using VOps = MMath<_Float16>;
    static constexpr int kParts = 1, kQ = 2, kP = 2, kSets = 1, kKeys = 64;
};
template <>
struct Px<q8_0_t> {
    using KOps = MMath<_Float16>;
    using VOps = MMath<__bf16>;
    static constexpr int kParts = 1, kQ = 2, kP = 3, kSets = 2, kKeys = 64;
};
template <>
struct Px<float> {
    using KOps = MMath<__bf16>;
    using VOps = MMath<__bf16>;
    static constexpr int kParts = 3, kQ = 3, kP = 3, kSets = 1, kKeys = 32;
};

constexpr int kPxGroups = kSharedWaves / 2;  // key groups: quarters of a stage

// One stage in LDS: rows of all key groups, `kParts` 16-bit images of K and V.
template <typename T>
struct PxStage {
    static constexpr int kRows = kPxGroups * Px<T>::kKeys;
    alignas(16) char k[Px<T>::kParts][kRows][128];
    alignas(16) char v[Px<T>::kParts][kRows][128];
    alignas(16) float kd[__is_same(T, q8_0_t) ? 2 : 1][__is_same(T, q8_0_t) ? kRows : 1];  // Q8_0 scales by dim half
    alignas(16) float vd[__is_same(T, q8_0_t) ? 2 : 1][__is_same(T, q8_0_t) ? kRows : 1];
};

__device__ __forceinline__ int px_k_at(int row, int chunk) { return (chunk ^ (row & 7)) << 4; }
__device__ __forceinline__ int px_v_at(int row, int chunk) { return (chunk ^ ((2 * row) & 7)) << 4; }

// This thread's share of a stage as fetched.
template <typename T>
struct PxRaw {
    static constexpr int N = __is_same(T, q8_0_t) ? 2 : 4;  // 16-byte chunks per tensor
    u32x4 k[N], v[N];
    unsigned kd, vd;  // Q8_0: threads 0 .. 255 the scale words of their row
};
template <typename T>
struct PxGeom {
    static constexpr int kPerRow = __is_same(T, float) ? 16 : __is_same(T, q8_0_t) ? 4 : 8;  // chunks per row
    static constexpr int kStep = 64 * kSharedWaves / kPerRow;                                              // rows per fetch
    static constexpr int kPages = PxStage<T>::kRows / kPageRows;                             // pages per stage
};

typedef unsigned u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

// Pool pages of a stage whose first page is logical page j0, as this wave
// fetches them (scalar loads, issued a stage before the rows).
template <typename T>
struct PxPages {
    static constexpr int N = __is_same(T, q8_0_t) ? 6 : 4;
    int page[N];
};
template <typename T>
__device__ __forceinline__ void px_pages(PxPages<T>& p, const const_i32_ptr table, int j0, int j_last, int wave) {
    using G = PxGeom<T>;
#pragma unroll
    for (int i = 0; i < PxPages<T>::N; ++i) {
        // rows of fetch i, then (Q8_0) of the scale words
        const int row0 = i < PxRaw<T>::N ? i * G::kStep + wave * 64 / G::kPerRow
                                         : 64 * (wave & 3) + kPageRows * (i - PxRaw<T>::N);
        p.page[i] = table[min(j0 + row0 / kPageRows, j_last)];
    }
}

template <typename T>
__device__ __forceinline__ void px_fetch(PxRaw<T>& r, const PagedAttnArgs& a, int h, const PxPages<T>& pages, int tid,
                                         unsigned& bad) {
    using G = PxGeom<T>;
    constexpr int HB = CacheFmt<T>::kHeadBytes;
    const int stride = a.n_kv_head * HB;
    auto base_of = [&](int i) {
        const int pg = pages.page[i];
        bad |= (unsigned)pg >= (unsigned)a.n_pages;
        return (size_t)min(max(pg, 0), a.n_pages - 1) * ((size_t)kPageRows * stride) + (size_t)h * HB;
    };
#pragma unroll
    for (int i = 0; i < PxRaw<T>::N; ++i) {
        const size_t base = base_of(i);
        const int row = (tid / G::kPerRow) % kPageRows;  // kStep is a multiple of a page's rows
        const size_t at = base + (size_t)row * stride + (tid % G::kPerRow) * 16;
        if constexpr (__is_same(T, q8_0_t)) {  // head rows are 4-byte aligned
            r.k[i] = *reinterpret_cast<const u32x4_a4*>(a.k_pages + at);
            r.v[i] = *reinterpret_cast<const u32x4_a4*>(a.v_pages + at);
        } else {
            r.k[i] = *reinterpret_cast<const u32x4*>(a.k_pages + at);
            r.v[i] = *reinterpret_cast<const u32x4*>(a.v_pages + at);
        }
    }
    if constexpr (__is_same(T, q8_0_t)) {
        // lanes of waves 0 .. 3: rows 64 wave + lane, four pages a wave (waves 4 .. 7 repeat them)
        const int row = tid & 255;
        size_t base = 0;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const size_t b = base_of(PxRaw<T>::N + p);
            base = (row & 63) / kPageRows == p ? b : base;
        }
        const size_t at = base + (size_t)(row % kPageRows) * stride + 64;
        r.kd = *reinterpret_cast<const unsigned*>(a.k_pages + at);
        r.vd = *reinterpret_cast<const unsigned*>(a.v_pages + at);
    }
}

// Three bf16 parts of two fp32 values (element 0 in the low half), cut bits: exact.
__device__ __forceinline__ void split3(float x, float y, unsigned (&w)[3]) {
    auto top = [](float v) { return __uint_as_float(__float_as_uint(v) & 0xFFFF0000u); };
    auto pair = [](float a, float b) { return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u); };
    w[0] = pair(x, y);
    const float x1 = x - top(x), y1 = y - top(y);
    w[1] = pair(x1, y1);
    w[2] = pair(x1 - top(x1), y1 - top(y1));
}
// Two fp16 parts (nearest, then the nearest to what is left).
__device__ __forceinline__ void split2(float x, float y, unsigned (&w)[3]) {
    w[0] = MMath<_Float16>::pack2(x, y);
    w[1] = MMath<_Float16>::pack2(x - MMath<_Float16>::lo(w[0]), y - MMath<_Float16>::hi(w[0]));
}

// Rows at or past `valid` of the stage: V is written as zeros (P is 0 there, and the row may hold anything).
template <typename T>
__device__ __forceinline__ void px_store(PxStage<T>& s, const PxRaw<T>& r, int valid, int tid) {
    using G = PxGeom<T>;
    const u32x4 zero = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < PxRaw<T>::N; ++i) {
        const int row = i * G::kStep + tid / G::kPerRow, q = tid % G::kPerRow;
        const u32x4 v = row < valid ? r.v[i] : zero;
        if constexpr (__is_same(T, float)) {
            const int half = 8 * (q & 1);
            unsigned k0[3], k1[3], v0[3], v1[3];
            split3(__uint_as_float(r.k[i][0]), __uint_as_float(r.k[i][1]), k0);
            split3(__uint_as_float(r.k[i][2]), __uint_as_float(r.k[i][3]), k1);
            split3(__uint_as_float(v[0]), __uint_as_float(v[1]), v0);
            split3(__uint_as_float(v[2]), __uint_as_float(v[3]), v1);
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                *reinterpret_cast<u32x2*>(&s.k[p][row][px_k_at(row, q / 2) + half]) = u32x2{k0[p], k1[p]};
                *reinterpret_cast<u32x2*>(&s.v[p][row][px_v_at(row, q / 2) + half]) = u32x2{v0[p], v1[p]};
            }
        } else if constexpr (__is_same(T, q8_0_t)) {  // 16 values: chunks 2 q, 2 q + 1
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const u32x2 ka = i8x4_to_f16(r.k[i][2 * c]), kb = i8x4_to_f16(r.k[i][2 * c + 1]);
                const u32x2 va = i8x4_to_bf16(v[2 * c]), vb = i8x4_to_bf16(v[2 * c + 1]);
                *reinterpret_cast<u32x4*>(&s.k[0][row][px_k_at(row, 2 * q + c)]) = u32x4{ka[0], ka[1], kb[0], kb[1]};
                *reinterpret_cast<u32x4*>(&s.v[0][row][px_v_at(row, 2 * q + c)]) = u32x4{va[0], va[1], vb[0], vb[1]};
            }
        } else {
            *reinterpret_cast<u32x4*>(&s.k[0][row][px_k_at(row, q)]) = r.k[i];
            *reinterpret_cast<u32x4*>(&s.v[0][row][px_v_at(row, q)]) = v;
        }
    }
    if constexpr (__is_same(T, q8_0_t)) {
        if (tid < PxStage<T>::kRows) {
            s.kd[0][tid] = half_bits_to_float(r.kd & 0xFFFFu);
            s.kd[1][tid] = half_bits_to_float(r.kd >> 16);
            const unsigned vd = tid < valid ? r.vd : 0u;
            s.vd[0][tid] = half_bits_to_float(vd & 0xFFFFu);
            s.vd[1][tid] = half_bits_to_float(vd >> 16);
        }
    }
}

// Whether part i of one operand meets part j of the other.
template <int NA, int NB>
constexpr bool px_pair(int i, int j) {
    return NA == 1 || NB == 1 || i + j <= 2;
}

// One wave's columns.
template <typename T>
struct PxCols {
    typename Px<T>::KOps::v8 q[2][2][Px<T>::kQ];  // [column block][dim half][part]
    float unscale[2];                             // fp16 operands: undoes the column's power of two
    f32x4 o[2][4];                                // block b, row r: dim 16 b + 4 g + r
    float m[2], l[2];
};

template <typename T>
__device__ __forceinline__ void px_load_q(PxCols<T>& c, int t, const float* p, float scale, int lane) {
    using X = Px<T>;
    const int g = lane >> 4;
    float x[2][8];
    float top = 0.f;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        float4 u = make_float4(0.f, 0.f, 0.f, 0.f), w = u;
        if (p) {
            u = *reinterpret_cast<const float4*>(p + 32 * m + 8 * g);
            w = *reinterpret_cast<const float4*>(p + 32 * m + 8 * g + 4);
        }
        const float y[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[m][e] = y[e] * scale;
            top = fmaxf(top, fabsf(x[m][e]));
        }
    }
    c.unscale[t] = 1.f;
    if constexpr (X::KOps::kScaleQ) {  // the column's largest value to [2^14, 2^15)
        top = max4_rows(top);
        const int e = min(max(14 - ((int)(__float_as_uint(top) >> 23) - 127), -126), 126);
        const float up = __uint_as_float((unsigned)(127 + e) << 23);
        c.unscale[t] = __uint_as_float((unsigned)(127 - e) << 23);
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[m][i] *= up;
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        u32x4 w[3];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            unsigned y[3] = {0, 0, 0};
            if constexpr (X::KOps::kScaleQ)
                split2(x[m][2 * i], x[m][2 * i + 1], y);
            else
                split3(x[m][2 * i], x[m][2 * i + 1], y);
#pragma unroll
            for (int k = 0; k < 3; ++k) w[k][i] = y[k];
        }
#pragma unroll
        for (int k = 0; k < X::kQ; ++k) c.q[t][m][k] = __builtin_bit_cast(typename X::KOps::v8, w[k]);
    }
}

// The wave's keys of one stage (rows row0 .. row0 + kKeys - 1, of which `valid` take part).
template <typename T>
__device__ __forceinline__ void px_attend(PxCols<T>& c, PxStage<T>& s, int row0, int valid, int lane) {
    using X = Px<T>;
    using KO = typename X::KOps;
    using VO = typename X::VOps;
    constexpr int KT = X::kKeys / 16;  // 16-key tiles
    constexpr bool Q8 = __is_same(T, q8_0_t);
    const int i = lane & 15, g = lane >> 4;
    f32x4 st[2][KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        const int row = row0 + 16 * kt + i;
        f32x4 acc[2][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) acc[t][0] = acc[t][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int kp = 0; kp < X::kParts; ++kp) {
                const auto kx = *reinterpret_cast<const typename KO::v8*>(&s.k[kp][row][px_k_at(row, 4 * m + g)]);
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int qp = 0; qp < X::kQ; ++qp)
                        if (px_pair<X::kParts, X::kQ>(kp, qp))
                            acc[t][Q8 ? m : 0] = KO::mfma32(kx, c.q[t][m][qp], acc[t][Q8 ? m : 0]);
            }
        if constexpr (Q8) {
            const f32x4 d0 = *reinterpret_cast<const f32x4*>(&s.kd[0][row0 + 16 * kt + 4 * g]);
            const f32x4 d1 = *reinterpret_cast<const f32x4*>(&s.kd[1][row0 + 16 * kt + 4 * g]);
#pragma unroll
            for (int t = 0; t < 2; ++t) st[t][kt] = (acc[t][0] * d0 + acc[t][1] * d1) * c.unscale[t];
        } else {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                st[t][kt] = acc[t][0];
                if constexpr (KO::kScaleQ) st[t][kt] *= c.unscale[t];
            }
        }
    }
    if (valid < X::kKeys) {
        asm volatile("");  // a branch: as selects the masks would cost every stage 48 instructions
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int t = 0; t < 2; ++t) st[t][kt][r] = 16 * kt + 4 * g + r < valid ? st[t][kt][r] : kNegInf;
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        float top = kNegInf;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
            top = fmaxf(top, fmaxf(fmaxf(st[t][kt][0], st[t][kt][1]), fmaxf(st[t][kt][2], st[t][kt][3])));
        if (__any(top > c.m[t] + kTau || c.m[t] == kNoMax)) {
            const float m1 = fmaxf(c.m[t], max4_rows(top));
            const float w = fast_exp2(c.m[t] - m1);
            c.m[t] = m1;
            c.l[t] *= w;
#pragma unroll
            for (int b = 0; b < 4; ++b) c.o[t][b] *= w;
        }
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
            for (int r = 0; r < 4; ++r) st[t][kt][r] = fast_exp2(st[t][kt][r] - c.m[t]);
            c.l[t] += (st[t][kt][0] + st[t][kt][1]) + (st[t][kt][2] + st[t][kt][3]);
        }
    }
    // 32 keys at a time: slots 8 g + e hold key 4 g + e of the first tile (e < 4) and of the second
#pragma unroll
    for (int ks = 0; ks < KT / 2; ++ks) {
        typename VO::v8 px[2][X::kSets][X::kP];
#pragma unroll
        for (int set = 0; set < X::kSets; ++set) {
            u32x4 w[2][3];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                f32x4 d = {VO::kPScale, VO::kPScale, VO::kPScale, VO::kPScale};
                if constexpr (Q8)
                    d = *reinterpret_cast<const f32x4*>(&s.vd[set][row0 + 32 * ks + 16 * half + 4 * g]);
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        float x = st[t][2 * ks + half][2 * r], y = st[t][2 * ks + half][2 * r + 1];
                        if constexpr (Q8 || VO::kPScale != 1.0f) x *= d[2 * r], y *= d[2 * r + 1];
                        unsigned z[3] = {0, 0, 0};
                        if constexpr (X::kP == 2)
                            split2(x, y, z);
                        else
                            split3(x, y, z);
#pragma unroll
                        for (int p = 0; p < X::kP; ++p) w[t][p][2 * half + r] = z[p];
                    }
            }
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int p = 0; p < X::kP; ++p) px[t][set][p] = __builtin_bit_cast(typename VO::v8, w[t][p]);
        }
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int vp = 0; vp < X::kParts; ++vp) {
                const int r0 = row0 + 32 * ks + 4 * g + (i >> 2), r1 = r0 + 16, chunk = 2 * b + ((i & 3) >> 1);
                const auto v0 = VO::read_tr(&s.v[vp][r0][px_v_at(r0, chunk) + 8 * (i & 1)]);
                const auto v1 = VO::read_tr(&s.v[vp][r1][px_v_at(r1, chunk) + 8 * (i & 1)]);
                const auto vx = VO::cat(v0, v1);
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int p = 0; p < X::kP; ++p)
                        if (px_pair<X::kParts, X::kP>(vp, p))
                            c.o[t][b] = VO::mfma32(vx, px[t][X::kSets == 2 ? b / 2 : 0][p], c.o[t][b]);
            }
    }
}

// The key groups' columns through LDS.
struct PxMerge {
    alignas(16) float o[kPxGroups][kSharedCols][kHeadDim + 4];
    float m[kPxGroups][kSharedCols], l[kPxGroups][kSharedCols];
};
template <typename T>
union PxLds {
    PxStage<T> stage[__is_same(T, float) ? 1 : 2];
    PxMerge merge;
};

template <typename T, typename ColPtr, typename Put>
__device__ __forceinline__ void px_run(const PagedAttnArgs& a, PxLds<T>& lds, const int32_t* table_, int h, int j0,
                                       int n_pages, int64_t rows, int n_cols, int tid, ColPtr col_ptr, Put put) {
    using X = Px<T>;
    using G = PxGeom<T>;
    constexpr int NB = __is_same(T, float) ? 1 : 2;
    const const_i32_ptr table = (const_i32_ptr)table_;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), kg = wave >> 1, cw = wave & 1;
    const int i = lane & 15, g = lane >> 4;
    const int n_stage = (n_pages + G::kPages - 1) / G::kPages, j_last = j0 + n_pages - 1;
    const int n_rows = (int)min((int64_t)n_pages * kPageRows, rows - (int64_t)j0 * kPageRows);  // of this run
    const bool busy = 32 * cw < n_cols;
    unsigned bad = 0;
    PxRaw<T> raw;
    PxPages<T> pages;
    px_pages<T>(pages, table, j0, j_last, wave);
    px_fetch<T>(raw, a, h, pages, tid, bad);
    px_pages<T>(pages, table, j0 + G::kPages, j_last, wave);
    PxCols<T> c;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        px_load_q<T>(c, t, col_ptr(32 * cw + 16 * t + i), a.qscale, lane);
        c.m[t] = kNoMax;
        c.l[t] = 0.f;
#pragma unroll
        for (int b = 0; b < 4; ++b) c.o[t][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    px_store<T>(lds.stage[0], raw, n_rows, tid);
    __syncthreads();
    for (int st = 0; st < n_stage; ++st) {
        PxStage<T>& cur = lds.stage[NB == 2 ? st & 1 : 0];
        const bool more = st + 1 < n_stage;
        if (more) {
            px_fetch<T>(raw, a, h, pages, tid, bad);
            px_pages<T>(pages, table, j0 + (st + 2) * G::kPages, j_last, wave);
        }
        const int valid = min(n_rows - st * PxStage<T>::kRows - kg * X::kKeys, X::kKeys);
        if (busy && valid > 0) px_attend<T>(c, cur, kg * X::kKeys, valid, lane);
        if (more) {
            if constexpr (NB == 1) __syncthreads();
            px_store<T>(lds.stage[NB == 2 ? (st + 1) & 1 : 0], raw, n_rows - (st + 1) * PxStage<T>::kRows, tid);
        }
        __syncthreads();
    }
    if (bad && lane == 0) atomicOr(a.err, 4);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int col = 32 * cw + 16 * t + i;
        const float l = sum4_rows(c.l[t]);
        if (g == 0) {
            lds.merge.m[kg][col] = c.m[t];
            lds.merge.l[kg][col] = l;
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            f32x4 o = c.o[t][b];
            if constexpr (X::VOps::kPScale != 1.0f) o *= 1.0f / X::VOps::kPScale;
            *reinterpret_cast<f32x4*>(&lds.merge.o[kg][col][16 * b + 4 * g]) = o;
        }
    }
    __syncthreads();
    // 8 threads a column, dims 4 d .. and 32 + 4 d ..
    const int col = tid >> 3, d = 4 * (tid & 7);
    if (col >= n_cols) return;
    float M = lds.merge.m[0][col], L = 0.f;
#pragma unroll
    for (int k = 1; k < kPxGroups; ++k) M = fmaxf(M, lds.merge.m[k][col]);
    f32x4 A = {0.f, 0.f, 0.f, 0.f}, B = A;
#pragma unroll
    for (int k = 0; k < kPxGroups; ++k) {
        const float x = fast_exp2(lds.merge.m[k][col] - M);
        L += x * lds.merge.l[k][col];
        A += x * *reinterpret_cast<const f32x4*>(&lds.merge.o[k][col][d]);
        B += x * *reinterpret_cast<const f32x4*>(&lds.merge.o[k][col][32 + d]);
    }
    put(col, d, M, L, A);
    put(col, 32 + d, M, L, B);
}

// Shared prefixes: workgroup (run of the prefix, kv head, block of 64 columns).
template <typename T>
__device__ __forceinline__ void prefix_body(const PagedAttnArgs& a) {
    __shared__ PxLds<T> lds;
    const int lane = threadIdx.x & 63, G = a.group;
    const int split = blockIdx.x, h = blockIdx.y;
    // the group whose column blocks hold this one
    Group grp = {0, 0, 0};
    int left = blockIdx.z;
    bool found = false;
    for (int g0 = 0; g0 < a.n_groups && !found; g0 += 64) {
        const Group g = group_at(a, g0 + lane);
        const int nb = (int)(((int64_t)(g.end - g.first) * G + kSharedCols - 1) / kSharedCols);
        int incl = nb;
        for (int m = 1; m < min(64, a.n_groups - g0); m *= 2) {
            const int o = __shfl_up(incl, m);
            if (lane >= m) incl += o;
        }
        const uint64_t b = __ballot(incl > left);
        const int at = b ? __builtin_ctzll(b) : 63;
        if (b) {
            grp.first = __builtin_amdgcn_readlane(g.first, at);
            grp.end = __builtin_amdgcn_readlane(g.end, at);
            grp.prefix = __builtin_amdgcn_readlane(g.prefix, at);
            found = true;
        }
        left -= __builtin_amdgcn_readlane(found ? incl - nb : incl, at);
    }
    const int64_t prefix = grp.prefix;
    if (!found || prefix == 0 || prefix > a.max_prefix) return;
    const int per = prefix_run_pages(a, prefix), j0 = split * per;
    const int n = min(per, (int)((prefix + kPageRows - 1) >> kPageShift) - j0);
    if (n <= 0) return;
    const int c0 = left * kSharedCols;                // this block's first column of the group
    const int cols = (grp.end - grp.first) * G - c0;  // columns from there on
    auto row_of = [&](int c) {
        const int s = (c0 + c) / G;
        return (int64_t)(grp.first + s) * a.n_head + h * G + (c0 + c - s * G);
    };
    px_run<T>(
        a, lds, a.block_table + (size_t)grp.first * a.max_pages, h, j0, n, prefix, cols, threadIdx.x,
        [&](int c) -> const float* { return c < cols ? a.q + row_of(c) * kHeadDim : nullptr; },
        [&](int c, int d, float M, float L, f32x4 A) { put_partial(a, row_of(c), split, d, M, L, A); });
}

// A sequence's own rows: workgroup (run of them, kv head, sequence).  FINISH:
// one run holds them all, and the workgroup merges the prefix's partials and
// writes the output; otherwise the run leaves one more partial.
template <typename T, bool FINISH>
__device__ __forceinline__ void tail_body(const PagedAttnArgs& a) {
    __shared__ MergeLds<kSharedWaves> lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int G = a.group, split = FINISH ? 0 : blockIdx.x, h = blockIdx.y, s = blockIdx.z;
    const int64_t row0 = (int64_t)s * a.n_head + h * G;
    const int col = lane & 15;
    Cols st;
    cols_init(st, col < G ? a.q + (row0 + col) * kHeadDim : nullptr, a.qscale, lane);
    const SharedSeq q = shared_seq(a, s, lane);
    const int64_t lo = q.prefix + (int64_t)split * a.tail_rows, hi = min(q.len, lo + a.tail_rows);
    if (!FINISH && (q.bad || lo >= hi)) return;
    if (!q.bad && lo < hi) {
        const int j0 = (int)(lo >> kPageShift), n = (int)((hi - 1) >> kPageShift) - j0 + 1;
        const int32_t* table = a.block_table + (size_t)s * a.max_pages;
        attend_run<T, kSharedWaves>(st, a, h, n, lo, hi, wave, lane, [&](int e, int& logical, int& page) {
            logical = j0 + e;
            page = table[logical];
            if (page < 0 || page >= a.n_pages) {
                atomicOr(a.err, 4);
                page = min(max(page, 0), a.n_pages - 1);
            }
        });
    }
    merge_waves<kSharedWaves>(st, lds, wave, lane, [&](int c, int d, float M, float L, f32x4 A) {
        if (c >= G) return;
        if constexpr (FINISH) {
            const int64_t per = (int64_t)prefix_run_pages(a, q.prefix) * kPageRows;
            const int n = q.bad || q.len == 0 ? 0 : (int)((q.prefix + per - 1) / per);
            const size_t at = (size_t)(row0 + c) * a.n_slots;
            const float* acc = a.ws + at * kHeadDim + d;
            const float2* ml =
                reinterpret_cast<const float2*>(a.ws + (size_t)a.n_seq * a.n_head * a.n_slots * kHeadDim) + at;
            for (int e0 = 0; e0 < n; e0 += 8) {  // eight partials at a time, their loads independent
                float2 x[8];
                f32x4 v[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int e = min(e0 + u, n - 1);
                    x[u] = ml[e];
                    v[u] = *reinterpret_cast<const f32x4*>(acc + (size_t)e * kHeadDim);
                }
                float m1 = M;
#pragma unroll
                for (int u = 0; u < 8; ++u) m1 = fmaxf(m1, x[u].x);
                const float f = fast_exp2(M - m1);
                L *= f;
                A *= f;
                M = m1;
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const float w = e0 + u < n ? fast_exp2(x[u].x - m1) : 0.f;
                    L += w * x[u].y;
                    A += w * v[u];
                }
            }
            A = finish_row(A, L);
            if (q.bad) {
                if (c == 0 && d == 0) atomicOr(a.err, 2);
                const float nan = __builtin_nanf("");
                A = f32x4{nan, nan, nan, nan};
            }
            *reinterpret_cast<f32x4*>(a.out + (row0 + c) * kHeadDim + d) = A;
        } else {
            put_partial(a, row0 + c, a.prefix_splits + split, d, M, L, A);
        }
    });
}

template <int WPR>
__device__ __forceinline__ void shared_merge_body(const PagedAttnArgs& a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = (int64_t)blockIdx.x * (kPagedWaves / WPR) + wave / WPR;
    if (row >= (int64_t)a.n_seq * a.n_head) return;
    const int s = __builtin_amdgcn_readfirstlane((int)(row / a.n_head));
    const SharedSeq q = shared_seq(a, s, lane);
    int n0 = 0, n1 = 0;
    if (!q.bad && q.len > 0) {
        const int64_t per = (int64_t)prefix_run_pages(a, q.prefix) * kPageRows;
        n0 = (int)((q.prefix + per - 1) / per);
        n1 = (int)((q.len - q.prefix + a.tail_rows - 1) / a.tail_rows);
    }
    float L;
    f32x4 y = merge_slots<WPR>(a, row, n0, a.prefix_splits, n1, wave % WPR, lane, L);
    if (wave % WPR || lane >= 16) return;
    y = finish_row(y, L);
    if (q.bad) {
        if (lane == 0) atomicOr(a.err, 2);
        const float nan = __builtin_nanf("");
        y = f32x4{nan, nan, nan, nan};
    }
    *reinterpret_cast<f32x4*>(a.out + row * kHeadDim + 4 * lane) = y;
}

}  // namespace

#define TMAC_PAGED_KERNELS(NAME, T)                                                                                    \
    extern "C" __global__ __launch_bounds__(256) void tmac_append_##NAME(AppendArgs a) { append_body<T>(a); }          \
    extern "C" __global__ __launch_bounds__(256) void tmac_page_bounds_##NAME(BoundsArgs a) { bounds_body<T>(a); }     \
    extern "C" __global__ __launch_bounds__(256) void tmac_selected_##NAME(PagedAttnArgs a) { selected_body<T>(a); }   \
    extern "C" __global__ __launch_bounds__(64 * kSharedWaves) void tmac_prefix_##NAME(PagedAttnArgs a) {               \
        prefix_body<T>(a);                                                                                             \
    }                                                                                                                  \
    extern "C" __global__ __launch_bounds__(64 * kSharedWaves) void tmac_tail_##NAME(PagedAttnArgs a) {                 \
        tail_body<T, false>(a);                                                                                        \
    }                                                                                                                  \
    extern "C" __global__ __launch_bounds__(64 * kSharedWaves) void tmac_tail_finish_##NAME(PagedAttnArgs a) {          \
        tail_body<T, true>(a);                                                                                         \
    }
TMAC_PAGED_KERNELS(f32, float)
TMAC_PAGED_KERNELS(bf16, __bf16)
TMAC_PAGED_KERNELS(f16, _Float16)
TMAC_PAGED_KERNELS(q8, q8_0_t)

#define TMAC_SCORE_KERNEL(GT) \
    extern "C" __global__ __launch_bounds__(256) void tmac_page_scores_g##GT(SelectArgs a) { score_body<GT>(a); }
TMAC_SCORE_KERNEL(1)
TMAC_SCORE_KERNEL(2)
TMAC_SCORE_KERNEL(3)
TMAC_SCORE_KERNEL(4)
TMAC_SCORE_KERNEL(5)
TMAC_SCORE_KERNEL(6)
TMAC_SCORE_KERNEL(7)
TMAC_SCORE_KERNEL(8)
extern "C" __global__ __launch_bounds__(kSelectThreads) void tmac_select_pages(SelectArgs a) { select_body(a); }
#define TMAC_MERGE_KERNELS(WPR)                                                                          \
    extern "C" __global__ __launch_bounds__(64 * kPagedWaves) void tmac_selected_merge_w##WPR(PagedAttnArgs a) { \
        selected_merge_body<WPR>(a);                                                                     \
    }                                                                                                    \
    extern "C" __global__ __launch_bounds__(64 * kPagedWaves) void tmac_shared_merge_w##WPR(PagedAttnArgs a) { \
        shared_merge_body<WPR>(a);                                                                       \
    }
TMAC_MERGE_KERNELS(1)
TMAC_MERGE_KERNELS(4)
