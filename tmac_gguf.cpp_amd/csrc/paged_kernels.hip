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
// Bound by memory: 18,095 fp16 rows of 14 query and 2 kv heads 32 us, 4.5 TB/s; 64
// rows 3.5 us, a launch and three dependent loads.
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
            load8(x, a.q + t * a.q_stride + (int64_t)h * kHeadDim + 4 * c);
            rope8(x, a.rope_cs + (size_t)pos * (kHeadDim / 2), c);
            store8(a.q_out + (t * nh + h) * kHeadDim + 4 * c, x);
        } else if (row >= 0) {
            const bool key = h < nh + kv;
            const int hk = key ? h - nh : h - nh - kv;
            load8(x, (key ? a.k + t * a.k_stride : a.v + t * a.v_stride) + (int64_t)hk * kHeadDim + 4 * c);
            if (key) rope8(x, a.rope_cs + (size_t)pos * (kHeadDim / 2), c);
            char* p = (key ? a.k_pages : a.v_pages) + (row * kv + hk) * HB + 4 * c * DB;
            put_row<T>(x, p, c, true);
        }
    }
}

// ---------------------------------------------------------------------------
// Page bounds.  One wave per (sequence, page, kv head): a slot of 8 lanes reads
// a row, 8 dims a lane, rows slot and slot + 8; the running max and min go
// over the slots with three lane exchanges.  Bound by memory: 8 sequences of up
// to 16,000 fp32 rows, 2 kv heads, 14 us, 3.8 TB/s.
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
    const int n = (int)min((int64_t)kPageRows, len - (int64_t)j * kPageRows);
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
// 2^-53).  max(q hi, q lo) = max(q, 0) hi + min(q, 0) lo, one of the products
// zero, so a score is a product of length 128 and runs on v_mfma_f64_4x4x4:
// four blocks of 4 pages x 4 heads x 4 dims in 16 cycles, where fp64 FMAs with
// a select and a sum over lanes took 37 us and this 21 (64 sequences of 2,048
// pages at most, 2 kv heads, 7 heads each; 20 with the steps dealt out, below).
//
// Lane l holds for a step of 16 pages: of the bounds, page 4 p + l % 4 (p =
// l / 4 % 4), dims 16 k .. 16 k + 15 (k = l / 16), product step t taking dim
// 16 k + t of every k; of the queries, head 4 hg + l % 4; of the sums, page
// 4 p + l / 16 and head 4 hg + l % 4.
// fp32 -> unsigned of the same order; NaN as +infinity.
__device__ __forceinline__ unsigned order_key(float x) {
    const unsigned u = x == x ? __float_as_uint(x) : 0x7F800000u;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int select_pages_of(const SelectArgs& a, int s) {  // -1: a bad length
    const int len = max(a.lengths[s], 0);
    return len > a.max_len ? -1 : (len >> kPageShift) + ((len & (kPageRows - 1)) != 0);
}

__device__ __forceinline__ double bf16_to_f64(unsigned w, int e) {
    return (double)__uint_as_float(e ? w & 0xFFFF0000u : w << 16);
}

template <int CTRL>
__device__ __forceinline__ unsigned dpp_u(unsigned x) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, false);
}

// Inclusive sum over the lanes of a wave.
__device__ __forceinline__ int wave_scan(int x, int lane) {
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        const int o = __shfl_up(x, m);
        if (lane >= m) x += o;
    }
    return x;
}

// One wave's steps g0, g0 + by, ... below g1 (16 pages each) of one (sequence,
// kv head) with n pages.  HG: groups of 4 query heads a pass takes.
template <int HG>
__device__ __forceinline__ void score_steps(const SelectArgs& a, int s, int h, int n, int g0, int g1, int by, int lane) {
    const int kv = a.n_kv_head, G = a.group, sk = s * kv + h;
    const int k = lane >> 4, p = (lane >> 2) & 3, i = lane & 3;
    const int32_t* table = a.block_table + (size_t)s * a.max_pages;
    unsigned* keys = a.keys + (size_t)sk * a.key_stride;
    auto page_at = [&](int g) {
        const int j = min(16 * g + 4 * p + i, n - 1), page = table[j];
        // the first and last pages are taken whatever their bounds
        if ((page < 0 || page >= a.n_pages) && k == 0 && j >= a.first && j < n - a.last) atomicOr(a.err, 4);
        return min(max(page, 0), a.n_pages - 1);
    };
    u32x4 hi[2], lo[2];
    auto fetch = [&](int page) {
        const uint16_t* b = a.bounds + ((size_t)page * kv + h) * (kBoundsBytes / 2) + 16 * k;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            hi[u] = *reinterpret_cast<const u32x4*>(b + 8 * u);
            lo[u] = *reinterpret_cast<const u32x4*>(b + kHeadDim + 8 * u);
        }
    };
    for (int head0 = 0; head0 < G; head0 += 4 * HG) {
        int page = page_at(g0);
        f32x4 q[HG][4];
#pragma unroll
        for (int hg = 0; hg < HG; ++hg) {
            const float* x =
                a.q + ((size_t)s * a.n_head + h * G + min(head0 + 4 * hg + i, G - 1)) * kHeadDim + 16 * k;
#pragma unroll
            for (int t = 0; t < 4; ++t) q[hg][t] = *reinterpret_cast<const f32x4*>(x + 4 * t);
        }
        fetch(page);
        page = page_at(min(g0 + by, g1 - 1));
        double up[HG][16], down[HG][16];
#pragma unroll
        for (int hg = 0; hg < HG; ++hg)
#pragma unroll
            for (int t = 0; t < 16; ++t) {
                const float x = q[hg][t / 4][t % 4];
                up[hg][t] = (double)fmaxf(x, 0.f);
                down[hg][t] = (double)fminf(x, 0.f);
            }
        for (int g = g0; g < g1; g += by) {
            const u32x4 vh[2] = {hi[0], hi[1]}, vl[2] = {lo[0], lo[1]};
            if (g + by < g1) {
                fetch(page);
                page = page_at(min(g + 2 * by, g1 - 1));
            }
            double sum[HG][2];  // two chains a head group
#pragma unroll
            for (int hg = 0; hg < HG; ++hg) sum[hg][0] = sum[hg][1] = 0.0;
#pragma unroll
            for (int t = 0; t < 16; ++t) {
                const double x = bf16_to_f64(vh[t / 8][t % 8 / 2], t % 2), y = bf16_to_f64(vl[t / 8][t % 8 / 2], t % 2);
#pragma unroll
                for (int hg = 0; hg < HG; ++hg) {
                    sum[hg][0] = __builtin_amdgcn_mfma_f64_4x4x4f64(x, up[hg][t], sum[hg][0], 0, 0, 0);
                    sum[hg][1] = __builtin_amdgcn_mfma_f64_4x4x4f64(y, down[hg][t], sum[hg][1], 0, 0, 0);
                }
            }
            unsigned best = 0;
#pragma unroll
            for (int hg = 0; hg < HG; ++hg)
                if (head0 + 4 * hg + i < G) best = max(best, order_key((float)(sum[hg][0] + sum[hg][1])));
            best = max(best, dpp_u<0xB1>(best));
            best = max(best, dpp_u<0x4E>(best));
            const int j = 16 * g + 4 * p + k;
            if (i == 0 && j < n) keys[j] = head0 ? max(keys[j], best) : best;
        }
    }
}

// Dealt out: the steps of all sequences in one row, cut into equal runs, a wave
// each, so that the lengths of a batch may differ as they like (64 sequences of
// 1,024 to 2,048 pages 21.5 -> 19.1 us).  A wave finds its run from the lengths
// itself.  Otherwise the grid has waves for each sequence.
template <int HG>
__device__ __forceinline__ void score_body(const SelectArgs& a) {
    const int lane = threadIdx.x & 63, kv = a.n_kv_head;
    const int wave = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * kPagedWaves + (threadIdx.x >> 6)));
    if (!a.dealt) {  // the kv heads of a sequence in turn, every waves / kv-th step
        const int s = blockIdx.y, h = wave % kv, n = select_pages_of(a, s), by = (int)(gridDim.x * kPagedWaves) / kv;
        const int steps = (n + 15) / 16, g0 = wave / kv;
        if (n > a.top && g0 < min(by, steps)) score_steps<HG>(a, s, h, n, g0, steps, by, lane);
        return;
    }
    constexpr int C = kScoreSeqs / 64;
    int steps[C], end[C], total = 0;  // this lane's sequences lane + 64 c: steps per kv head, where their steps end
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int s = lane + 64 * c, n = s < a.n_seq ? select_pages_of(a, s) : 0;
        steps[c] = n > a.top ? (n + 15) / 16 : 0;
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
        if (64 * c >= a.n_seq) {
            end[c] = total;
            continue;
        }
        end[c] = total + wave_scan(steps[c] * kv, lane);
        total = __builtin_amdgcn_readlane(end[c], 63);
    }
    const int64_t waves = gridDim.x * kPagedWaves;
    int at = (int)(total * (int64_t)wave / waves);
    const int stop = (int)(total * (int64_t)(wave + 1) / waves);
    while (at < stop) {
        int s = 0, m = 0, e = 0;  // the sequence that holds step `at`
#pragma unroll
        for (int c = C - 1; c >= 0; --c) {
            const uint64_t b = __ballot(end[c] > at);
            if (b) {
                const int l = __builtin_ctzll(b);
                s = 64 * c + l;
                m = __builtin_amdgcn_readlane(steps[c], l);
                e = __builtin_amdgcn_readlane(end[c], l);
            }
        }
        const int x = at - (e - m * kv), h = x / m, g0 = x - h * m, g1 = min(m, g0 + stop - at);
        score_steps<HG>(a, s, h, select_pages_of(a, s), g0, g1, 1, lane);
        at += g1 - g0;
    }
}

// The top pages of one (sequence, kv head), ascending.  The top-th largest key
// is found two bits at a time from the highest bit in which the keys differ:
// three candidates are counted at once, and a count of exactly top ends the
// search.  Then the keys above it and the first of those equal to it
// are written in page order.  The keys stay in registers (the first kSelectRegs
// a thread; longer sequences read the rest again).  What bounds it is the
// latency of a turn: the lanes' counts, their sum, a barrier and the waves' counts,
// 1,200 cycles (64 sequences of up to 2,048 pages, 2 kv heads: 10.4 us).
constexpr int kSelectRegs = 8;  // 64 of them at most 1,023: counts of ten bits

// Maximum over a wave, and sum over each row of 16 lanes, without the LDS crossbar.
__device__ __forceinline__ unsigned wave_max_u(unsigned x) {
    x = max(x, dpp_u<0xB1>(x));
    x = max(x, dpp_u<0x4E>(x));
    x = max(x, dpp_u<0x141>(x));
    x = max(x, dpp_u<0x128>(x));
    const auto p = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max((unsigned)p[0], (unsigned)p[1]);
    const auto q = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return max((unsigned)q[0], (unsigned)q[1]);
}
__device__ __forceinline__ unsigned row_sum_u(unsigned x) {
    x += dpp_u<0xB1>(x);
    x += dpp_u<0x4E>(x);
    x += dpp_u<0x141>(x);
    return x + dpp_u<0x128>(x);
}

__device__ __forceinline__ unsigned wave_sum_u(unsigned x) {
    x = row_sum_u(x);
    const auto p = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = (unsigned)p[0] + (unsigned)p[1];
    const auto q = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return (unsigned)q[0] + (unsigned)q[1];
}

template <int NT>
__device__ __forceinline__ void select_body(const SelectArgs& a) {
    constexpr int NW = NT / 64;
    static_assert(NW <= 16, "a row of lanes sums the waves' counts");
    __shared__ unsigned s_count[2][3][16];  // by turn, candidate, wave
    __shared__ unsigned s_range[2][16];
    __shared__ unsigned s_scan[kSelectRegs * NW];  // by round, wave: pages above the threshold << 16 | pages equal to it
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int sk = blockIdx.x, s = sk / a.n_kv_head;
    const int n = select_pages_of(a, s);
    int32_t* out = a.selected + (size_t)sk * a.top;
    if (n < 0 && tid == 0) atomicOr(a.err, 2);
    if (n <= a.top) {
        for (int i = tid; i < a.top; i += NT) out[i] = i < n ? i : -1;
        return;
    }
    const unsigned* keys = a.keys + (size_t)sk * a.key_stride;
    const int rounds = (n + NT - 1) / NT, held = min(rounds, kSelectRegs);
    // Key of page j: forced pages above every score (a score's key is at most that of +infinity), none below.
    auto key_at = [&](int j) {
        const unsigned k = j < n ? keys[j] : 0u;
        return j >= n ? 0u : j < a.first || j >= n - a.last ? 0xFFFFFFFFu : k;
    };
    unsigned k[kSelectRegs];
#pragma unroll
    for (int r = 0; r < kSelectRegs; ++r) k[r] = r < held ? key_at(r * NT + tid) : 0u;
    if (tid < 96) s_count[tid / 48][tid / 16 % 3][tid % 16] = 0;
    // The highest bit in which the scored keys differ (as the largest key and the largest complement of one).
    unsigned hi = 0u, nlo = 0u;
    auto range = [&](unsigned x) {
        if (x && x != 0xFFFFFFFFu) hi = max(hi, x), nlo = max(nlo, ~x);
    };
#pragma unroll
    for (int r = 0; r < kSelectRegs; ++r) range(k[r]);
    for (int r = kSelectRegs; r < rounds; ++r) range(key_at(r * NT + tid));
    hi = wave_max_u(hi);
    nlo = wave_max_u(nlo);
    if (lane == 0) s_range[0][wave] = hi, s_range[1][wave] = nlo;
    __syncthreads();
    hi = wave_max_u(s_range[0][lane % NW]);
    const unsigned lo = ~wave_max_u(s_range[1][lane % NW]);
    // n > top >= first + last, so there are scored keys; the top-th largest key is one of them or, with top = first +
    // last, the threshold stays above them all.
    const unsigned top = (unsigned)a.top;
    unsigned prefix;  // no fewer than top keys are >= prefix; in the end the top-th largest key, or all >= are taken
    if (a.first + a.last == a.top) {
        prefix = 0xFFFFFFFFu;
    } else {
        int bits = lo == hi ? 0 : 32 - __builtin_clz(lo ^ hi);
        bits = (bits + 1) & ~1;
        prefix = bits >= 32 ? 0u : lo >> bits << bits;
        prefix = __builtin_amdgcn_readfirstlane(prefix);
        bits = __builtin_amdgcn_readfirstlane(bits);
        for (int turn = 0; bits > 0; turn ^= 1) {
            bits -= 2;
            // Counted a lane and summed over the wave as one word (at most 64 kSelectRegs each): a ballot each would
            // wait for its comparison before the next, 1,450 cycles a turn.
            const unsigned c1 = prefix | 1u << bits, c2 = prefix | 2u << bits, c3 = prefix | 3u << bits;
            unsigned packed = 0;
#pragma unroll
            for (int r = 0; r < kSelectRegs; ++r)
                packed += (k[r] >= c1 ? 1u : 0u) + (k[r] >= c2 ? 1u << 10 : 0u) + (k[r] >= c3 ? 1u << 20 : 0u);
            packed = wave_sum_u(packed);
            unsigned c[3] = {packed & 1023u, packed >> 10 & 1023u, packed >> 20};
            for (int r = kSelectRegs; r < rounds; ++r) {
                const unsigned x = key_at(r * NT + tid);
                c[0] += __popcll(__ballot(x >= c1));
                c[1] += __popcll(__ballot(x >= c2));
                c[2] += __popcll(__ballot(x >= c3));
            }
            if (lane == 0) {
#pragma unroll
                for (int d = 0; d < 3; ++d) s_count[turn][d][wave] = c[d];
            }
            __syncthreads();
            const unsigned t = row_sum_u(s_count[turn][min(lane / 16, 2)][lane % 16]);
            const unsigned t0 = __builtin_amdgcn_readlane(t, 0), t1 = __builtin_amdgcn_readlane(t, 16),
                           t2 = __builtin_amdgcn_readlane(t, 32);
            const int d = t2 >= top ? 3 : t1 >= top ? 2 : t0 >= top ? 1 : 0;
            prefix |= (unsigned)d << bits;
            if ((d == 3 ? t2 : d == 2 ? t1 : d == 1 ? t0 : 0) == top) break;  // exactly the keys >= prefix
        }
    }
    // Taken: keys > prefix, then the first of those equal to it, as many as are left.  (After an exact end the equal
    // ones are just those.)  Of the held rounds every wave leaves its counts; a scan over (round, wave) places them.
    int places[kSelectRegs];  // this thread's pages before it in its wave and round: above << 16 | equal
#pragma unroll
    for (int r = 0; r < kSelectRegs; ++r) {
        if (r >= held) break;
        const uint64_t bg = __ballot(k[r] > prefix), be = __ballot(k[r] == prefix), below = (1ull << lane) - 1;
        places[r] = __popcll(bg & below) << 16 | __popcll(be & below);
        if (lane == 0) s_scan[r * NW + wave] = (unsigned)__popcll(bg) << 16 | (unsigned)__popcll(be);
    }
    __syncthreads();
    // entries 2 lane, 2 lane + 1 of the scan (NW * kSelectRegs <= 128)
    const unsigned e0 = 2 * lane < held * NW ? s_scan[2 * lane] : 0u;
    const unsigned e1 = 2 * lane + 1 < held * NW ? s_scan[2 * lane + 1] : 0u;
    unsigned incl = e0 + e1;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        const unsigned o = __shfl_up(incl, m);
        if (lane >= m) incl += o;
    }
    const unsigned all = __builtin_amdgcn_readlane(incl, 63), before = incl - e0 - e1;
    // keys above the threshold: those of the rounds that are not held count too
    unsigned above = all >> 16;
    if (rounds > kSelectRegs) {
        unsigned more = 0;
        for (int r = kSelectRegs; r < rounds; ++r) more += __popcll(__ballot(key_at(r * NT + tid) > prefix));
        if (lane == 0) s_count[0][0][wave] = more;
        __syncthreads();
        above += __builtin_amdgcn_readlane(row_sum_u(s_count[0][0][lane % 16]), 0);
    }
    const int left = (int)(top - above);
    auto place = [&](unsigned x, int j, int g, int e) {
        if (j < n && (x > prefix || (x == prefix && e < left))) out[g + min(e, left)] = j;
    };
#pragma unroll
    for (int r = 0; r < kSelectRegs; ++r) {
        if (r >= held) break;
        const int at = r * NW + wave;
        const unsigned b = __builtin_amdgcn_readlane(before, at / 2) + (at % 2 ? __builtin_amdgcn_readlane(e0, at / 2) : 0u);
        const unsigned p = b + (unsigned)places[r];
        place(k[r], r * NT + tid, (int)(p >> 16), (int)(p & 0xFFFFu));
    }
    int b_gt = (int)(all >> 16), b_eq = (int)(all & 0xFFFFu);  // pages before a round that is not held
    for (int r = kSelectRegs; r < rounds; ++r) {
        const unsigned x = key_at(r * NT + tid);
        const uint64_t bg = __ballot(x > prefix), be = __ballot(x == prefix), below = (1ull << lane) - 1;
        __syncthreads();
        if (lane == 0) s_scan[wave] = (unsigned)__popcll(bg) << 16 | (unsigned)__popcll(be);
        __syncthreads();
        unsigned b = 0, sum = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            if (w < wave) b += s_scan[w];
            sum += s_scan[w];
        }
        place(x, r * NT + tid, b_gt + (int)(b >> 16) + __popcll(bg & below), b_eq + (int)(b & 0xFFFFu) + __popcll(be & below));
        b_gt += (int)(sum >> 16);
        b_eq += (int)(sum & 0xFFFFu);
    }
}

// Short lists: scores and selection of one list in one workgroup.
template <int HG>
__device__ __forceinline__ void select_short_body(const SelectArgs& a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sk = blockIdx.x, s = sk / a.n_kv_head, n = select_pages_of(a, s), steps = (n + 15) / 16;
    if (n > a.top && wave < steps) score_steps<HG>(a, s, sk - s * a.n_kv_head, n, wave, steps, kPagedWaves, lane);
    __syncthreads();
    select_body<64 * kPagedWaves>(a);
}

// ---------------------------------------------------------------------------
// Decode attention, common parts.  A column is one query head of one sequence;
// scores and sums are kept transposed, S^T (keys x columns) and O^T (dims x
// columns), so that a lane owns columns and the softmax is lane-local but for a
// rare exchange.
//
// bf16, fp16 and Q8_0 rows run on 16-bit MFMA, every fp32 operand carried by
// 16-bit parts that together hold it (three bf16 all 24 bits, two fp16 to
// 2^-23), so the result keeps fp32 accuracy:
//   cache   K, V        q            P            products, Q.K and P.V
//   bf16    exact       3 bf16       3 bf16       3, 3
//   fp16    exact       2 fp16       2 fp16       2, 2
//   Q8_0    int8 exact  2 fp16       3 bf16 x 2   2, 3 (scales on S and on P)
//   fp32    3 bf16      3 bf16       3 bf16       6, 6 (parts i + j <= 2)
// Of fp32 rows the products i + j > 2 are left out.  Parts are cut, not rounded,
// so these have the sign of the whole product; they are at most 2^-21 of it, and
// 0.7 x 2^-24 of it on average.
// (Two bf16 parts of P, 2^-18, left 2e-6 of the output's norm.)  fp32 rows are
// split where many columns share them (prefixes) and go to fp32 MFMA where only
// one group of query heads reads them.
template <typename T>
struct Parts;
template <>
struct Parts<__bf16> {
    using KOps = MMath<__bf16>;
    using VOps = MMath<__bf16>;
    static constexpr int kCache = 1, kQ = 3, kP = 3, kSets = 1;
};
template <>
struct Parts<_Float16> {
    using KOps = MMath<_Float16>;
    using VOps = MMath<_Float16>;
    static constexpr int kCache = 1, kQ = 2, kP = 2, kSets = 1;
};
template <>
struct Parts<q8_0_t> {
    using KOps = MMath<_Float16>;
    using VOps = MMath<__bf16>;
    static constexpr int kCache = 1, kQ = 2, kP = 3, kSets = 2;
};
template <>
struct Parts<float> {
    using KOps = MMath<__bf16>;
    using VOps = MMath<__bf16>;
    static constexpr int kCache = 3, kQ = 3, kP = 3, kSets = 1;
};

// Whether part i of one operand meets part j of the other.
template <int NA, int NB>
constexpr bool parts_meet(int i, int j) {
    return NA == 1 || NB == 1 || i + j <= 2;
}

// Three bf16 parts of two fp32 values (element 0 in the low half), cut bits: exact.
__device__ __forceinline__ unsigned top_pair(float x, float y) {
    return __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
}
__device__ __forceinline__ void split3(float x, float y, unsigned (&w)[3]) {
    auto top = [](float v) { return __uint_as_float(__float_as_uint(v) & 0xFFFF0000u); };
    w[0] = top_pair(x, y);
    const float x1 = x - top(x), y1 = y - top(y);
    w[1] = top_pair(x1, y1);
    w[2] = top_pair(x1 - top(x1), y1 - top(y1));
}
// Q and P: KP parts; fp16: two, each the nearest.  What remains of a value is
// taken with a mask and a subtraction, which issue beside a product (4 in the 32
// cycles of one cost 1 more): a dot product with (-1, 0) does it in one
// instruction, but runs on the matrix unit's time, 8 cycles and a product's wait.
template <typename M, int KP>
__device__ __forceinline__ void split(float x, float y, unsigned (&w)[3]) {
    if constexpr (M::kScaleQ) {
        static_assert(KP == 2, "fp16: 22 bits in two parts");
        w[0] = M::pack2(x, y);
        const f16x2 v = __builtin_bit_cast(f16x2, w[0]);
        w[1] = M::pack2(x - (float)v[0], y - (float)v[1]);
    } else {
        static_assert(KP == 3, "bf16: 24 bits in three parts");
        split3(x, y, w);
    }
}

constexpr float kNoMax = -__FLT_MAX__;  // running maximum of a column that has met no key

typedef float f32x16 __attribute__((ext_vector_type(16)));

// MFMA shapes.  Cols columns, lane groups g of Cols lanes; a product contracts
// Depth values, 8 a lane group.  In an accumulator lane (column, g) holds rows
// row(r) + 4 g, four in a run.
struct Mfma16 {
    static constexpr int kCols = 16, kDepth = 32, kAcc = 4;
    using Acc = f32x4;
    template <typename M>
    __device__ static Acc mul(typename M::v8 a, typename M::v8 b, Acc c) { return M::mfma32(a, b, c); }
    __device__ static float top(float x) { return max4_rows(x); }
    __device__ static float sum(float x) { return sum4_rows(x); }
};
struct Mfma32 {
    static constexpr int kCols = 32, kDepth = 16, kAcc = 16;
    using Acc = f32x16;
    template <typename M>
    __device__ static Acc mul(typename M::v8 a, typename M::v8 b, Acc c) {
        if constexpr (M::kScaleQ)
            return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    __device__ static float top(float x) { return xor_max<32>(x); }
    __device__ static float sum(float x) { return xor_sum<32>(x); }
};

// One wave's columns on shape S.  Operand of q: depth block m, part p: lane
// (column, g) the dims kDepth m + 8 g + 0..7.  Sums: dim block b of 64 / kCols.
template <typename T, typename S>
struct Cols {
    static constexpr int kDepthBlocks = kHeadDim / S::kDepth, kDimBlocks = kHeadDim / S::kCols;
    typename Parts<T>::KOps::v8 q[kDepthBlocks][Parts<T>::kQ];
    typename S::Acc o[kDimBlocks];
    float unscale;  // fp16 operands: undoes the column's power of two
    float m, l;     // m: kNoMax until a key was met; l: this lane's keys
    float base;     // what is subtracted from the scores: m, 0 before the first key
};

template <typename Acc>
__device__ __forceinline__ Acc acc_of(float x) {
    Acc a;
#pragma unroll
    for (int r = 0; r < (int)(sizeof(Acc) / 4); ++r) a[r] = x;
    return a;
}

// The raw query values of a lane (p null: an unused column), and empty columns made of them.
template <typename T, typename S>
struct RawQ {
    f32x4 x[Cols<T, S>::kDepthBlocks][2];
};
template <typename T, typename S>
__device__ __forceinline__ void load_q(RawQ<T, S>& r, const float* p, int lane) {
    const int g = lane / S::kCols;
#pragma unroll
    for (int m = 0; m < Cols<T, S>::kDepthBlocks; ++m)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            r.x[m][i] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (p) r.x[m][i] = *reinterpret_cast<const f32x4*>(p + S::kDepth * m + 8 * g + 4 * i);
        }
}
template <typename T, typename S>
__device__ __forceinline__ void cols_init(Cols<T, S>& c, const RawQ<T, S>& raw, float scale) {
    using KO = typename Parts<T>::KOps;
    constexpr int MB = Cols<T, S>::kDepthBlocks;
    float x[MB][8];
    float top = 0.f;
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[m][e] = raw.x[m][e / 4][e % 4] * scale;
            top = fmaxf(top, fabsf(x[m][e]));
        }
    c.unscale = 1.f;
    if constexpr (KO::kScaleQ) {  // the column's largest value to [2^14, 2^15)
        top = S::top(top);
        const int e = min(max(14 - ((int)(__float_as_uint(top) >> 23) - 127), -126), 126);
        const float up = __uint_as_float((unsigned)(127 + e) << 23);
        c.unscale = __uint_as_float((unsigned)(127 - e) << 23);
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[m][i] *= up;
    }
#pragma unroll
    for (int m = 0; m < MB; ++m) {
        u32x4 w[3];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            unsigned y[3] = {0, 0, 0};
            split<KO, Parts<T>::kQ>(x[m][2 * i], x[m][2 * i + 1], y);
#pragma unroll
            for (int k = 0; k < 3; ++k) w[k][i] = y[k];
        }
#pragma unroll
        for (int k = 0; k < Parts<T>::kQ; ++k) c.q[m][k] = __builtin_bit_cast(typename KO::v8, w[k]);
    }
    c.m = kNoMax;
    c.l = c.base = 0.f;
#pragma unroll
    for (int b = 0; b < Cols<T, S>::kDimBlocks; ++b) c.o[b] = acc_of<typename S::Acc>(0.f);
}

// Scores minus base of one tile of S::kCols keys.  key(m, p): the K operand,
// depth block m, part p.  kd0 / kd1 (Q8_0): the keys' scales by dim half.
// bf16 operands are summed onto -base.
template <typename T, typename S, typename Key>
__device__ __forceinline__ typename S::Acc score_tile(const Cols<T, S>& c, const float* kd0, const float* kd1, int g,
                                                      Key key) {
    using P = Parts<T>;
    using KO = typename P::KOps;
    constexpr bool Q8 = __is_same(T, q8_0_t), FROM_BASE = !Q8 && !KO::kScaleQ;
    constexpr int MB = Cols<T, S>::kDepthBlocks;
    typename S::Acc acc[2] = {acc_of<typename S::Acc>(FROM_BASE ? -c.base : 0.f), acc_of<typename S::Acc>(0.f)};
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
        for (int kp = 0; kp < P::kCache; ++kp) {
            const auto kx = key(m, kp);
#pragma unroll
            for (int qp = 0; qp < P::kQ; ++qp)
                if (parts_meet<P::kCache, P::kQ>(kp, qp)) {
                    const int half = Q8 && 2 * m >= MB;
                    acc[half] = S::template mul<KO>(kx, c.q[m][qp], acc[half]);
                }
        }
    if constexpr (Q8) {
#pragma unroll
        for (int r4 = 0; r4 < S::kAcc / 4; ++r4) {
            const f32x4 d0 = *reinterpret_cast<const f32x4*>(kd0 + 8 * r4 + 4 * g);
            const f32x4 d1 = *reinterpret_cast<const f32x4*>(kd1 + 8 * r4 + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                acc[0][4 * r4 + r] = __builtin_fmaf(
                    __builtin_fmaf(acc[1][4 * r4 + r], d1[r], acc[0][4 * r4 + r] * d0[r]), c.unscale, -c.base);
        }
    } else if constexpr (!FROM_BASE) {
#pragma unroll
        for (int r = 0; r < S::kAcc; ++r) acc[0][r] = __builtin_fmaf(acc[0][r], c.unscale, -c.base);
    }
    return acc[0];
}

// Scores minus base of NT tiles -> weights, online: the base is raised only
// when a score exceeds it by more than kTau.
template <typename S, int NB, int NT>
__device__ __forceinline__ void softmax_step(float& m, float& l, float& base, typename S::Acc (&o)[NB],
                                             typename S::Acc (&st)[NT]) {
    // Whether any score is over the base by more than kTau, as integers: their order is that of the floats where it
    // matters (above a positive bound), and a maximum of them needs no quieting of NaN.
    int over = INT32_MIN;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < S::kAcc; ++r) over = max(over, (int)__float_as_uint(st[t][r]));
    if (__any(over > (int)__float_as_uint(kTau) || m == kNoMax)) {
        float top = kNegInf;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < S::kAcc; ++r) top = fmaxf(top, st[t][r]);
        const float m1 = fmaxf(m, base + S::top(top));
        const float b1 = m1 == kNoMax ? 0.f : m1, shift = b1 - base;
        const float w = fast_exp2(m - m1);
        m = m1;
        base = b1;
        l *= w;
#pragma unroll
        for (int b = 0; b < NB; ++b) o[b] *= w;
#pragma unroll
        for (int t = 0; t < NT; ++t) st[t] -= shift;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < S::kAcc; ++r) {
            st[t][r] = fast_exp2(st[t][r]);
            sum += st[t][r];
        }
        l += sum;
    }
}

// 16-byte chunks of a 128-byte LDS row are XORed with the row, K by row & 7, V
// by 2 row & 7, so that operand reads touch all banks.
__device__ __forceinline__ int k_chunk(int row, int chunk) { return (chunk ^ (row & 7)) << 4; }
__device__ __forceinline__ int v_chunk(int row, int chunk) { return (chunk ^ ((2 * row) & 7)) << 4; }

// O^T += V^T . P^T over one product depth of keys.  w0, w1: four weights each of
// the lane's keys r + 4 g and of those kDepth / 2 rows behind; v: the V image's
// first row of the block (a multiple of 4 rows), part images part_bytes apart;
// vd0 / vd1 (Q8_0): the keys' scales by dim half.  V is read back transposed:
// with ds_read_b64_tr_b16 the 16 lanes of a group point at 4 rows x 32 bytes,
// and each receives 4 consecutive keys of one dim.
template <typename T, typename S>
__device__ __forceinline__ void values_step(Cols<T, S>& c, f32x4 w0, f32x4 w1, char* v, int part_bytes,
                                            const float* vd0, const float* vd1, int lane) {
    using P = Parts<T>;
    using VO = typename P::VOps;
    constexpr bool Q8 = __is_same(T, q8_0_t);
    constexpr int kBack = S::kDepth / 2;
    const int i = lane & 15, g = lane / S::kCols;
    typename VO::v8 px[P::kSets][P::kP];
#pragma unroll
    for (int set = 0; set < P::kSets; ++set) {
        u32x4 w[3];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            f32x4 x = half ? w1 : w0;
            if constexpr (Q8)
                x *= *reinterpret_cast<const f32x4*>((set ? vd1 : vd0) + kBack * half + 4 * g);
            else if constexpr (VO::kPScale != 1.0f)
                x *= VO::kPScale;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                unsigned z[3] = {0, 0, 0};
                split<VO, P::kP>(x[2 * r], x[2 * r + 1], z);
#pragma unroll
                for (int p = 0; p < P::kP; ++p) w[p][2 * half + r] = z[p];
            }
        }
#pragma unroll
        for (int p = 0; p < P::kP; ++p) px[set][p] = __builtin_bit_cast(typename VO::v8, w[p]);
    }
    const int sub = (lane / 16) % (S::kCols / 16);  // which 16 dims of a 32-dim block this lane's group reads
#pragma unroll
    for (int b = 0; b < Cols<T, S>::kDimBlocks; ++b)
#pragma unroll
        for (int vp = 0; vp < P::kCache; ++vp) {
            const int r0 = 4 * g + (i >> 2), r1 = r0 + kBack;
            const int chunk = S::kCols / 8 * b + 2 * sub + ((i & 3) >> 1);
            char* p = v + vp * part_bytes + 8 * (i & 1);
            const auto vx = VO::cat(VO::read_tr(p + r0 * 128 + v_chunk(r0, chunk)),
                                    VO::read_tr(p + r1 * 128 + v_chunk(r1, chunk)));
#pragma unroll
            for (int pp = 0; pp < P::kP; ++pp)
                if (parts_meet<P::kCache, P::kP>(vp, pp))
                    c.o[b] = S::template mul<VO>(vx, px[P::kSets == 2 ? b * S::kCols / 32 : 0][pp], c.o[b]);
        }
}

// ---------------------------------------------------------------------------
// Own rows: one group of query heads (up to 16 columns) over a run of pages,
// which its wave alone reads.  What bounds it is the rows' bytes; a wave holds
// one step of pages while the next is in flight (three or four ahead were slower).
// 64 sequences of 128 listed bf16 pages on 2 kv heads: 18.4 us, 3.7 TB/s.
typedef unsigned u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u32x2_a4 __attribute__((ext_vector_type(2), aligned(4)));

// 16-bit and Q8_0 rows: two pages a step, 32 keys.  K is read as the MFMA operand
// it is, V through LDS (a buffer of the wave's own, no barrier), where it comes
// back transposed.  fp32 MFMA on widened rows, 16 times the cycles for a
// product, took 20.2 us for 64 x 128 bf16 pages of 2 kv heads, and a wave 1,000
// cycles a page where it waits on its own products.
template <typename T>
struct Own {
    using S = Mfma16;
    using State = Cols<T, S>;
    using RawQuery = RawQ<T, S>;
    static constexpr int kTiles = 2;
    static constexpr bool Q8 = __is_same(T, q8_0_t);
    struct Tile {
        u32x4 k[Q8 ? 1 : 2], v[Q8 ? 1 : 2];
        unsigned kd, vd;  // Q8_0: the scale words of row lane % 16
    };
    struct Lds {
        alignas(16) char v[32][128];
        alignas(16) float kd[Q8 ? 2 : 1][Q8 ? 32 : 1], vd[Q8 ? 2 : 1][Q8 ? 32 : 1];
    };
    __device__ static void query(RawQuery& q, const float* p, int lane) { load_q<T, S>(q, p, lane); }
    __device__ static void init(State& st, const RawQuery& q, float scale) { cols_init<T, S>(st, q, scale); }

    // kp / vp: row 0 of the page's head; stride: bytes between rows (64 bits: 15 rows of 559,241 fp32 kv heads pass 2^31).
    __device__ static void fetch(Tile& t, const char* kp, const char* vp, size_t stride, int lane) {
        const int i = lane & 15, g = lane >> 4;
        if constexpr (Q8) {  // dims 8 g .. and 32 + 8 g .. of key i; 16 values of row lane / 4
            const u32x2 a = *reinterpret_cast<const u32x2_a4*>(kp + i * stride + 8 * g);
            const u32x2 b = *reinterpret_cast<const u32x2_a4*>(kp + i * stride + 32 + 8 * g);
            t.k[0] = u32x4{a[0], a[1], b[0], b[1]};
            t.kd = *reinterpret_cast<const unsigned*>(kp + i * stride + 64);
            t.v[0] = *reinterpret_cast<const u32x4_a4*>(vp + (lane >> 2) * stride + 16 * (lane & 3));
            t.vd = *reinterpret_cast<const unsigned*>(vp + i * stride + 64);
        } else {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                t.k[m] = *reinterpret_cast<const u32x4*>(kp + i * stride + 64 * m + 16 * g);
                t.v[m] = *reinterpret_cast<const u32x4*>(vp + (8 * m + (lane >> 3)) * stride + 16 * (lane & 7));
            }
        }
    }
    // Keys lo[u] .. hi[u] - 1 of page u take part.
    __device__ static void attend(State& st, const Tile (&t)[kTiles], const int (&lo)[kTiles], const int (&hi)[kTiles],
                                  Lds& lds, int lane) {
        using KO = typename Parts<T>::KOps;
        const int i = lane & 15, g = lane >> 4;
        const u32x4 zero = {0, 0, 0, 0};
        const bool full = lo[0] <= 0 && lo[1] <= 0 && hi[0] >= kPageRows && hi[1] >= kPageRows;
#pragma unroll
        for (int u = 0; u < 2; ++u) {  // a row outside may hold anything: zeros
            auto in = [&](int r) { return full || (r >= lo[u] && r < hi[u]); };
            if constexpr (Q8) {
                const int r = lane >> 2, q = lane & 3, row = 16 * u + r;
                const u32x4 v = in(r) ? t[u].v[0] : zero;
                const u32x2 a = i8x4_to_bf16(v[0]), b = i8x4_to_bf16(v[1]), c = i8x4_to_bf16(v[2]),
                            d = i8x4_to_bf16(v[3]);
                *reinterpret_cast<u32x4*>(&lds.v[row][v_chunk(row, 2 * q)]) = u32x4{a[0], a[1], b[0], b[1]};
                *reinterpret_cast<u32x4*>(&lds.v[row][v_chunk(row, 2 * q + 1)]) = u32x4{c[0], c[1], d[0], d[1]};
                if (lane < 16) {
                    const unsigned vd = in(i) ? t[u].vd : 0u;
                    lds.kd[0][16 * u + i] = half_bits_to_float(t[u].kd & 0xFFFFu);
                    lds.kd[1][16 * u + i] = half_bits_to_float(t[u].kd >> 16);
                    lds.vd[0][16 * u + i] = half_bits_to_float(vd & 0xFFFFu);
                    lds.vd[1][16 * u + i] = half_bits_to_float(vd >> 16);
                }
            } else {
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    const int r = 8 * m + (lane >> 3), row = 16 * u + r;
                    *reinterpret_cast<u32x4*>(&lds.v[row][v_chunk(row, lane & 7)]) = in(r) ? t[u].v[m] : zero;
                }
            }
        }
        f32x4 w[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
            w[u] = score_tile<T, S>(st, &lds.kd[0][Q8 ? 16 * u : 0], &lds.kd[Q8 ? 1 : 0][Q8 ? 16 * u : 0], g,
                                    [&](int m, int) {
                                        if constexpr (Q8) {
                                            const u32x2 a = i8x4_to_f16(t[u].k[0][2 * m]),
                                                        b = i8x4_to_f16(t[u].k[0][2 * m + 1]);
                                            return __builtin_bit_cast(typename KO::v8, u32x4{a[0], a[1], b[0], b[1]});
                                        } else {
                                            return __builtin_bit_cast(typename KO::v8, t[u].k[m]);
                                        }
                                    });
        if (!full) {
            asm volatile("");  // a branch, not selects
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) w[u][r] = 4 * g + r >= lo[u] && 4 * g + r < hi[u] ? w[u][r] : kNegInf;
        }
        softmax_step<S>(st.m, st.l, st.base, st.o, w);
        values_step<T, S>(st, w[0], w[1], &lds.v[0][0], 0, lds.vd[0], lds.vd[Q8 ? 1 : 0], lane);
    }
    // This lane's sums of column lane % 16, ready to merge: dims 16 b + 4 g + 0..3.
    static constexpr int dim(int b, int g) { return 16 * b + 4 * g; }
    __device__ static f32x4 sums(const State& st, int b) {
        constexpr float k = Parts<T>::VOps::kPScale;
        return k != 1.0f ? st.o[b] * (1.0f / k) : st.o[b];
    }
};

// fp32 rows: one page a step on v_mfma_f32_16x16x4_f32, straight from registers.
// Step (m, e) of K contracts the four dims 32 m + 8 g + e, g = 0..3.  The
// accumulator S^T leaves keys 4 g + r in lane group g, so step r of V contracts
// the keys 4 g + r from the same registers; row i of block b is dim 4 i + b, so
// lane (i, g) reads V of key 4 g + r as the four dims 4 i + 0..3.
template <>
struct Own<float> {
    using S = Mfma16;
    static constexpr int kTiles = 1;
    struct State {
        float q[16];
        f32x4 o[4];  // block b, row r: dim 16 g + 4 r + b
        float m, l, base;
    };
    struct RawQuery {
        f32x4 x[4];
    };
    struct Tile {
        f32x4 k[4], v[4];
    };
    struct Lds {};
    __device__ static void query(RawQuery& q, const float* p, int lane) {
        const int g = lane >> 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            q.x[j] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (p) q.x[j] = *reinterpret_cast<const f32x4*>(p + 32 * (j / 2) + 8 * g + 4 * (j % 2));
        }
    }
    __device__ static void init(State& st, const RawQuery& q, float scale) {
#pragma unroll
        for (int j = 0; j < 16; ++j) st.q[j] = q.x[j / 4][j % 4] * scale;
        st.m = kNoMax;
        st.l = st.base = 0.f;
#pragma unroll
        for (int b = 0; b < 4; ++b) st.o[b] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    __device__ static void fetch(Tile& t, const char* kp, const char* vp, size_t stride, int lane) {
        const int i = lane & 15, g = lane >> 4;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            t.k[j] = *reinterpret_cast<const f32x4*>(kp + i * stride + 128 * (j / 2) + 32 * g + 16 * (j % 2));
#pragma unroll
        for (int r = 0; r < 4; ++r) t.v[r] = *reinterpret_cast<const f32x4*>(vp + (4 * g + r) * stride + 16 * i);
    }
    __device__ static void attend(State& st, const Tile (&tiles)[1], const int (&lo)[1], const int (&hi)[1], Lds&,
                                  int lane) {
        const Tile& t = tiles[0];
        const int g = lane >> 4;
        const bool full = lo[0] <= 0 && hi[0] >= kPageRows;
        // two sums: a chain of 16 dependent products would wait on itself
        f32x4 w[1] = {f32x4{-st.base, -st.base, -st.base, -st.base}}, w1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            w[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(t.k[e / 4][e % 4], st.q[e], w[0], 0, 0, 0);
            w1 = __builtin_amdgcn_mfma_f32_16x16x4f32(t.k[2 + e / 4][e % 4], st.q[8 + e], w1, 0, 0, 0);
        }
        w[0] += w1;
        auto in = [&](int r) { return full || (4 * g + r >= lo[0] && 4 * g + r < hi[0]); };
        if (!full) {
            asm volatile("");
#pragma unroll
            for (int r = 0; r < 4; ++r) w[0][r] = in(r) ? w[0][r] : kNegInf;
        }
        softmax_step<S>(st.m, st.l, st.base, st.o, w);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int b = 0; b < 4; ++b)  // a row outside may hold anything
                st.o[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(in(r) ? t.v[r][b] : 0.f, w[0][r], st.o[b], 0, 0, 0);
    }
    static constexpr int dim(int b, int g) { return 16 * g + 4 * b; }
    __device__ static f32x4 sums(const State& st, int b) { return f32x4{st.o[0][b], st.o[1][b], st.o[2][b], st.o[3][b]}; }
};

// LDS of a workgroup of NW waves on own rows: the waves' buffers, then the merge.
template <int NW>
struct MergeLds {
    alignas(16) float o[NW][16][kHeadDim + 4];
    float m[NW][16], l[NW][16];
};
template <typename T, int NW>
union OwnLds {
    typename Own<T>::Lds own[NW];
    MergeLds<NW> merge;
    __device__ OwnLds() {}
};

// A run of pages.  look(e, logical, page) gives entry e (0 <= e < n) its page of
// the pool (checked, in range) and its logical page index (-1: skipped); rows
// row_lo .. row_hi - 1 of the sequence take part.  The NW waves take the
// entries in turn, kTiles at once; a wave looks up 64 of its entries at a time,
// one a lane.
template <typename T, int NW, typename Look>
__device__ __forceinline__ void attend_run(typename Own<T>::State& st, const PagedAttnArgs& a, int h, int n,
                                           int64_t row_lo, int64_t row_hi, typename Own<T>::Lds& lds, int wave,
                                           int lane, Look look) {
    using O = Own<T>;
    constexpr int HB = CacheFmt<T>::kHeadBytes, KT = O::kTiles;
    const size_t stride = (size_t)a.n_kv_head * HB, page_bytes = kPageRows * stride;
    const int steps = ((n + KT - 1) / KT - wave + NW - 1) / NW;  // this wave's
    for (int s0 = 0; s0 < steps; s0 += 64 / KT) {
        const int cnt = min(64 / KT, steps - s0);
        int logical = -1, page = 0;
        const int e = ((s0 + lane / KT) * NW + wave) * KT + lane % KT;
        if (lane < cnt * KT && e < n) look(e, logical, page);
        typename O::Tile t[2][KT];
        auto fetch = [&](typename O::Tile (&x)[KT], int step) {
#pragma unroll
            for (int u = 0; u < KT; ++u) {
                const size_t at = (size_t)__builtin_amdgcn_readlane(page, KT * step + u) * page_bytes + (size_t)h * HB;
                O::fetch(x[u], a.k_pages + at, a.v_pages + at, stride, lane);
            }
        };
        fetch(t[0], 0);
        for (int step = 0; step < cnt; step += 2) {
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                if (step + d < cnt) {
                    if (step + d + 1 < cnt) fetch(t[1 - d], step + d + 1);
                    int lo[KT], hi[KT], any = 0;
#pragma unroll
                    for (int u = 0; u < KT; ++u) {
                        const int j = __builtin_amdgcn_readlane(logical, KT * (step + d) + u);
                        const int64_t r0 = (int64_t)j * kPageRows;
                        lo[u] = (int)max((int64_t)0, min(row_lo - r0, (int64_t)kPageRows));
                        hi[u] = j < 0 ? 0 : (int)max((int64_t)0, min(row_hi - r0, (int64_t)kPageRows));
                        any |= hi[u] > lo[u];
                    }
                    if (any) O::attend(st, t[d], lo, hi, lds, lane);
                }
            }
        }
    }
}

// Merges the NW waves through LDS and hands every column's maximum, sum and
// four dims to put(column, first dim, m, l, acc): one call a thread of the first
// 256 (16 columns x 16 dim quads).
template <typename T, int NW, typename Put>
__device__ __forceinline__ void merge_waves(const typename Own<T>::State& st, MergeLds<NW>& lds, int wave, int lane,
                                            Put put) {
    const int i = lane & 15, g = lane >> 4;
    const float l = sum4_rows(st.l);
    __syncthreads();  // the buffers of all waves are done with
    if (g == 0) {
        lds.m[wave][i] = st.m;
        lds.l[wave][i] = l;
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) *reinterpret_cast<f32x4*>(&lds.o[wave][i][Own<T>::dim(b, g)]) = Own<T>::sums(st, b);
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
template <typename T, int NW>
__device__ __forceinline__ void selected_body(const PagedAttnArgs& a) {
    __shared__ OwnLds<T, NW> lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kv = a.n_kv_head, G = a.group;
    const int split = blockIdx.x % a.n_slots, sk = blockIdx.x / a.n_slots, s = sk / kv, h = sk - s * kv;
    const int len = a.lengths[s];
    const int e0 = split * a.per_split, n = min(a.per_split, a.top - e0);
    const int32_t* list = a.selected + (size_t)sk * a.top + e0;
    const int32_t* table = a.block_table + (size_t)s * a.max_pages;
    const int64_t row0 = (int64_t)s * a.n_head + h * G;
    const int col = lane & 15;
    typename Own<T>::RawQuery raw;
    typename Own<T>::State st;
    Own<T>::query(raw, col < G ? a.q + (row0 + col) * kHeadDim : nullptr, lane);
    Own<T>::init(st, raw, a.qscale);
    attend_run<T, NW>(st, a, h, n, 0, len, lds.own[wave], wave, lane, [&](int e, int& logical, int& page) {
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
    merge_waves<T, NW>(st, lds.merge, wave, lane, [&](int c, int d, float M, float L, f32x4 A) {
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

// Blocks of 64 columns a group has.
__device__ __forceinline__ int blocks_of(const PagedAttnArgs& a, const Group& g) {
    return (int)(((int64_t)(g.end - g.first) * a.group + kSharedCols - 1) / kSharedCols);
}

// Runs that every prefix is cut into: as many as give each workgroup of the
// prefix kernel's grid one unit, with n_blocks blocks in all, and at most those
// there are slots for.  Pages of one run of a prefix of `prefix` rows.
__device__ __forceinline__ int prefix_runs(const PagedAttnArgs& a, int n_blocks) {
    return max(1, min(a.prefix_splits, a.prefix_groups / max(1, n_blocks * a.n_kv_head)));
}
__device__ __forceinline__ int run_pages(int64_t prefix, int runs) {
    const int n = (int)((prefix + kPageRows - 1) >> kPageShift);
    return max(1, (n + runs - 1) / runs);
}

// A sequence's rows: [0, prefix) through its group's first sequence, [prefix,
// len) through its own pages.  Its group is the last one that holds it.
struct SharedSeq {
    int64_t prefix, len;
    int64_t own;  // first row that the sequence reads itself
    int leader;   // the group's first sequence
    int slots;    // partials that the prefix left
    bool bad;   // a length or prefix outside what the launch covers
};
__device__ __forceinline__ SharedSeq shared_seq(const PagedAttnArgs& a, int s, int lane) {
    SharedSeq r;
    r.len = max(a.lengths[s], 0);
    r.prefix = 0;
    r.leader = s;
    int n_blocks = 0;
    for (int g0 = 0; g0 < a.n_groups; g0 += 64) {
        const Group g = group_at(a, g0 + lane);
        const uint64_t b = __ballot(s >= g.first && s < g.end);
        if (b) {
            r.prefix = __builtin_amdgcn_readlane(g.prefix, 63 - __clzll(b));
            r.leader = __builtin_amdgcn_readlane(g.first, 63 - __clzll(b));
        }
        n_blocks += (int)__builtin_amdgcn_readfirstlane(wave_sum_u((unsigned)blocks_of(a, g)));
    }
    r.bad = r.len > 0 && (r.prefix > a.max_prefix || r.len < r.prefix || r.len - r.prefix > a.max_tail ||
                          r.len > (int64_t)a.max_pages * kPageRows);
    const int64_t per = (int64_t)run_pages(r.prefix, prefix_runs(a, min(n_blocks, a.prefix_blocks))) * kPageRows;
    r.own = a.prefix_splits ? r.prefix : 0;
    r.slots = r.bad || r.len == 0 ? 0 : (int)((r.own + per - 1) / per);
    return r;
}

// ---------------------------------------------------------------------------
// Shared prefix.  A workgroup of 8 waves takes 64 columns, (sequence, query
// head) pairs of one group and kv head, over a run of the prefix: wave (kg, cw)
// the columns 32 cw .. 32 cw + 31 and, of every stage, the keys of quarter kg,
// on v_mfma_f32_32x32x16.  What bounds it is the issue of products and of the
// softmax beside them, about 3,000 cycles for a wave's 64 keys x 32 columns.
// A stage's K and V rows go to LDS once, fetched one stage ahead, and feed both
// column waves: 16-bit rows directly, fp32 and Q8_0 ones through registers, where
// they are converted.  96 sequences of 14 heads on 2 behind 16,384 rows: bf16 26.4
// us, 214 TFLOP/s (641 of parts); of the 6,000 cycles of a stage half are products;
// fp16 25.2, Q8_0 36.5, fp32, six products each, 50 us.
template <typename T>
constexpr int kPxKeys = __is_same(T, float) ? 32 : 64;  // keys a wave takes of a stage
constexpr int kPxGroups = kSharedWaves / 2;             // key groups: quarters of a stage

// One stage in LDS: rows of all key groups, Parts::kCache 16-bit images of K and V.
template <typename T>
struct PxStage {
    static constexpr int kRows = kPxGroups * kPxKeys<T>;
    static constexpr bool Q8 = __is_same(T, q8_0_t);
    alignas(16) char k[Parts<T>::kCache][kRows][128];
    alignas(16) char v[Parts<T>::kCache][kRows][128];
    alignas(16) float kd[Q8 ? 2 : 1][Q8 ? kRows : 1];  // Q8_0 scales by dim half
    alignas(16) float vd[Q8 ? 2 : 1][Q8 ? kRows : 1];
};

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

// 16-bit rows need no conversion and go from memory to LDS without registers
// between (64 lanes x 16 bytes, 8 rows, to consecutive LDS): the XOR of a row's
// chunks is in the address that a lane reads.  Rows at or past `valid` of the
// stage are past the end of the descriptor and come as zeros.  The loads are
// counted with vmcnt; px_landed() before the barrier that opens the stage.
__device__ __forceinline__ void load_lds16(u32x4 descriptor, unsigned offset, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 ::"s"(lds), "v"(offset), "s"(descriptor) : "memory", "m0");
}
__device__ __forceinline__ void px_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
template <typename T>
__device__ __forceinline__ void px_direct(PxStage<T>& s, const PagedAttnArgs& a, int h, const PxPages<T>& pages,
                                          int valid, int wave, int lane, unsigned& bad) {
    using G = PxGeom<T>;
    const unsigned stride = a.n_kv_head * 128u;
    const int row = 8 * wave + lane / 8, slot = lane & 7;  // + 64 i: the same place in its page, the same XOR
    const unsigned at = row % kPageRows * stride, ko = at + k_chunk(row, slot), vo = at + v_chunk(row, slot);
#pragma unroll
    for (int i = 0; i < PxRaw<T>::N; ++i) {
        const int pg = pages.page[i], r0 = i * G::kStep + 8 * wave, rows = valid - r0 / kPageRows * kPageRows;
        bad |= (unsigned)pg >= (unsigned)a.n_pages;
        const size_t base =
            (size_t)min(max(pg, 0), a.n_pages - 1) * ((size_t)kPageRows * stride) + (size_t)h * 128;
        const unsigned bytes = rows > 0 ? (min(rows, kPageRows) - 1) * stride + 128 : 0;
        auto load = [&](const char* pool, unsigned offset, char* to) {
            const uint64_t p = reinterpret_cast<uint64_t>(pool + base);
            load_lds16(u32x4{(unsigned)p, (unsigned)(p >> 32) & 0xFFFFu, bytes, 0x00020000u}, offset,
                       (unsigned)reinterpret_cast<size_t>((__attribute__((address_space(3))) char*)to));
        };
        load(a.k_pages, ko, &s.k[0][r0][0]);
        load(a.v_pages, vo, &s.v[0][r0][0]);
    }
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
                *reinterpret_cast<u32x2*>(&s.k[p][row][k_chunk(row, q / 2) + half]) = u32x2{k0[p], k1[p]};
                *reinterpret_cast<u32x2*>(&s.v[p][row][v_chunk(row, q / 2) + half]) = u32x2{v0[p], v1[p]};
            }
        } else if constexpr (__is_same(T, q8_0_t)) {  // 16 values: chunks 2 q, 2 q + 1
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const u32x2 ka = i8x4_to_f16(r.k[i][2 * c]), kb = i8x4_to_f16(r.k[i][2 * c + 1]);
                const u32x2 va = i8x4_to_bf16(v[2 * c]), vb = i8x4_to_bf16(v[2 * c + 1]);
                *reinterpret_cast<u32x4*>(&s.k[0][row][k_chunk(row, 2 * q + c)]) = u32x4{ka[0], ka[1], kb[0], kb[1]};
                *reinterpret_cast<u32x4*>(&s.v[0][row][v_chunk(row, 2 * q + c)]) = u32x4{va[0], va[1], vb[0], vb[1]};
            }
        } else {
            *reinterpret_cast<u32x4*>(&s.k[0][row][k_chunk(row, q)]) = r.k[i];
            *reinterpret_cast<u32x4*>(&s.v[0][row][v_chunk(row, q)]) = v;
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

// The wave's keys of one stage (rows row0 .. row0 + kPxKeys - 1, of which `valid` take part).
template <typename T>
__device__ __forceinline__ void px_attend(Cols<T, Mfma32>& c, PxStage<T>& s, int row0, int valid,
                                          int lane) {
    using S = Mfma32;
    using KO = typename Parts<T>::KOps;
    constexpr bool Q8 = PxStage<T>::Q8;
    constexpr int KT = kPxKeys<T> / 32;  // 32-key tiles
    const int i = lane & 31, g = lane >> 5;
    f32x16 st[KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        const int first = row0 + 32 * kt, row = first + i;
        st[kt] = score_tile<T, S>(c, &s.kd[0][Q8 ? first : 0], &s.kd[Q8 ? 1 : 0][Q8 ? first : 0], g,
                                  [&](int m, int p) {
                                      return *reinterpret_cast<const typename KO::v8*>(
                                          &s.k[p][row][k_chunk(row, 2 * m + g)]);
                                  });
    }
    if (valid < kPxKeys<T>) {
        asm volatile("");  // a branch: as selects the masks would cost every stage 48 instructions
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                st[kt][r] = 32 * kt + 8 * (r / 4) + 4 * g + r % 4 < valid ? st[kt][r] : kNegInf;
    }
    softmax_step<S>(c.m, c.l, c.base, c.o, st);
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // 16 keys at a time: the lane's weights 8 h + 0..3 and 8 h + 4..7
            const int first = row0 + 32 * kt + 16 * h;
            const f32x4 w0 = {st[kt][8 * h], st[kt][8 * h + 1], st[kt][8 * h + 2], st[kt][8 * h + 3]};
            const f32x4 w1 = {st[kt][8 * h + 4], st[kt][8 * h + 5], st[kt][8 * h + 6], st[kt][8 * h + 7]};
            values_step<T, S>(c, w0, w1, &s.v[0][first][0], sizeof(s.v[0]), &s.vd[0][Q8 ? first : 0],
                              &s.vd[Q8 ? 1 : 0][Q8 ? first : 0], lane);
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
    using G = PxGeom<T>;
    constexpr int NB = __is_same(T, float) ? 1 : 2;
    constexpr bool Direct = CacheFmt<T>::kHeadBytes == 128;
    const const_i32_ptr table = (const_i32_ptr)table_;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), kg = wave >> 1, cw = wave & 1;
    const int i = lane & 31, g = lane >> 5;
    const int n_stage = (n_pages + G::kPages - 1) / G::kPages, j_last = j0 + n_pages - 1;
    const int n_rows = (int)min((int64_t)n_pages * kPageRows, rows - (int64_t)j0 * kPageRows);  // of this run
    const bool busy = 32 * cw < n_cols;
    unsigned bad = 0;
    PxRaw<T> raw;
    PxPages<T> pages;
    Cols<T, Mfma32> c;
    px_pages<T>(pages, table, j0, j_last, wave);
    {
        RawQ<T, Mfma32> q;
        load_q<T, Mfma32>(q, col_ptr(32 * cw + i), lane);
        if constexpr (Direct) px_direct<T>(lds.stage[0], a, h, pages, n_rows, wave, lane, bad);
        else px_fetch<T>(raw, a, h, pages, tid, bad);
        px_pages<T>(pages, table, j0 + G::kPages, j_last, wave);
        cols_init<T, Mfma32>(c, q, a.qscale);
    }
    if constexpr (Direct) px_landed();
    else px_store<T>(lds.stage[0], raw, n_rows, tid);
    __syncthreads();
    for (int st = 0; st < n_stage; ++st) {
        PxStage<T>& cur = lds.stage[NB == 2 ? st & 1 : 0];
        PxStage<T>& next = lds.stage[NB == 2 ? (st + 1) & 1 : 0];
        const bool more = st + 1 < n_stage;
        const int after = n_rows - (st + 1) * PxStage<T>::kRows;
        if (more) {
            if constexpr (Direct) px_direct<T>(next, a, h, pages, after, wave, lane, bad);
            else px_fetch<T>(raw, a, h, pages, tid, bad);
            px_pages<T>(pages, table, j0 + (st + 2) * G::kPages, j_last, wave);
        }
        const int valid = min(n_rows - st * PxStage<T>::kRows - kg * kPxKeys<T>, kPxKeys<T>);
        if (busy && valid > 0) px_attend<T>(c, cur, kg * kPxKeys<T>, valid, lane);
        if (more) {
            if constexpr (NB == 1) __syncthreads();
            if constexpr (!Direct) px_store<T>(next, raw, after, tid);
        }
        if constexpr (Direct) px_landed();
        __syncthreads();
    }
    if (bad && lane == 0) atomicOr(a.err, 4);
    {
        const int col = 32 * cw + i;
        const float l = Mfma32::sum(c.l);
        if (g == 0) {
            lds.merge.m[kg][col] = c.m;
            lds.merge.l[kg][col] = l;
        }
        constexpr float k = 1.0f / Parts<T>::VOps::kPScale;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4)
                *reinterpret_cast<f32x4*>(&lds.merge.o[kg][col][32 * b + 8 * r4 + 4 * g]) =
                    f32x4{c.o[b][4 * r4], c.o[b][4 * r4 + 1], c.o[b][4 * r4 + 2], c.o[b][4 * r4 + 3]} * k;
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

// Shared prefixes: a unit is (run of the prefix, kv head, block of 64 columns).
// Consecutive workgroups go to the eight XCDs in turn, and the blocks of a run
// read the same rows: every XCD takes a contiguous eighth of the (run, kv head,
// block) order, so that a row is read into one L2, or two, and not all eight.
// How many blocks there are follows from the groups; a workgroup takes further
// units where there are more than the grid.  None starts for nothing: one that
// finds no work still waits for a CU with its LDS free (131 KB for 16-bit rows, 139
// for Q8_0, 98 for fp32), and 160 of them behind 240 others took 10 us.
template <typename T>
__device__ __forceinline__ void prefix_body(const PagedAttnArgs& a) {
    __shared__ PxLds<T> lds;
    const int lane = threadIdx.x & 63, G = a.group;
    // The blocks there are: 64 groups at a time, one a lane, their blocks summed.
    const Group first64 = group_at(a, lane);
    const int incl64 = wave_scan(blocks_of(a, first64), lane);
    int n_blocks = __builtin_amdgcn_readlane(incl64, 63);
    for (int g0 = 64; g0 < a.n_groups; g0 += 64)
        n_blocks += __builtin_amdgcn_readlane(wave_scan(blocks_of(a, group_at(a, g0 + lane)), lane), 63);
    n_blocks = min(n_blocks, a.prefix_blocks);
    const int runs = prefix_runs(a, n_blocks), n_units = runs * a.n_kv_head * n_blocks, per_xcd = (n_units + kXcds - 1) / kXcds;
    for (int at_xcd = (int)(blockIdx.x / kXcds); at_xcd < per_xcd; at_xcd += (int)(gridDim.x / kXcds)) {
        const int unit = (int)(blockIdx.x % kXcds) * per_xcd + at_xcd;
        if (unit >= n_units) break;
        const int run = unit / n_blocks, h = run % a.n_kv_head, split = run / a.n_kv_head;
        // the group that holds this block
        int left = unit - run * n_blocks;
        Group grp = first64;
        int incl = incl64;
        for (int g0 = 0; g0 < a.n_groups; g0 += 64) {
            if (g0) {
                grp = group_at(a, g0 + lane);
                incl = wave_scan(blocks_of(a, grp), lane);
            }
            const uint64_t b = __ballot(incl > left);
            if (b) {
                const int at = __builtin_ctzll(b);
                left -= __builtin_amdgcn_readlane(incl - blocks_of(a, grp), at);
                grp.first = __builtin_amdgcn_readlane(grp.first, at);
                grp.end = __builtin_amdgcn_readlane(grp.end, at);
                grp.prefix = __builtin_amdgcn_readlane(grp.prefix, at);
                break;
            }
            left -= __builtin_amdgcn_readlane(incl, 63);
        }
        const int64_t prefix = __builtin_amdgcn_readfirstlane(grp.prefix);
        if (prefix == 0 || prefix > a.max_prefix) continue;
        const int per = run_pages(prefix, runs), j0 = split * per;
        const int n = min(per, (int)((prefix + kPageRows - 1) >> kPageShift) - j0);
        if (n <= 0) continue;
        const int first = __builtin_amdgcn_readfirstlane(grp.first), end = __builtin_amdgcn_readfirstlane(grp.end);
        const int c0 = left * kSharedCols;        // this block's first column of the group
        const int cols = (end - first) * G - c0;  // columns from there on
        auto row_of = [&](int c) {
            const int s = (c0 + c) / G;
            return (int64_t)(first + s) * a.n_head + h * G + (c0 + c - s * G);
        };
        px_run<T>(
            a, lds, a.block_table + (size_t)first * a.max_pages, h, j0, n, prefix, cols, threadIdx.x,
            [&](int c) -> const float* { return c < cols ? a.q + row_of(c) * kHeadDim : nullptr; },
            [&](int c, int d, float M, float L, f32x4 A) { put_partial(a, row_of(c), split, d, M, L, A); });
        __syncthreads();  // the stage buffers of the next unit are those of this one's merge
    }
}

// A sequence's own rows: workgroup (run of them, kv head, sequence).  FINISH:
// one run holds them all, and the workgroup merges the prefix's partials and
// writes the output; otherwise the run leaves one more partial.
template <typename T, int NW, bool FINISH>
__device__ __forceinline__ void tail_body(const PagedAttnArgs& a) {
    __shared__ OwnLds<T, NW> lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int G = a.group, split = FINISH ? 0 : blockIdx.x, h = blockIdx.y, s = blockIdx.z;
    const int64_t row0 = (int64_t)s * a.n_head + h * G;
    const int col = lane & 15;
    typename Own<T>::RawQuery raw;
    typename Own<T>::State st;
    Own<T>::query(raw, col < G ? a.q + (row0 + col) * kHeadDim : nullptr, lane);
    const SharedSeq q = shared_seq(a, s, lane);
    Own<T>::init(st, raw, a.qscale);
    const int64_t lo = q.own + (int64_t)split * a.tail_rows, hi = min(q.len, lo + a.tail_rows);
    if (!FINISH && (q.bad || lo >= hi)) return;
    // rows of the prefix through the first sequence's table, then its own
#pragma unroll 1
    for (int part = lo < q.prefix ? 0 : 1; part < 2; ++part) {
        const int64_t r0 = part ? max(lo, q.prefix) : lo, r1 = part ? hi : min(hi, q.prefix);
        if (q.bad || r0 >= r1) continue;
        const int j0 = (int)(r0 >> kPageShift), n = (int)((r1 - 1) >> kPageShift) - j0 + 1;
        const int32_t* table = a.block_table + (size_t)(part ? s : q.leader) * a.max_pages;
        attend_run<T, NW>(st, a, h, n, r0, r1, lds.own[wave], wave, lane, [&](int e, int& logical, int& page) {
            logical = j0 + e;
            page = table[logical];
            if (page < 0 || page >= a.n_pages) {
                atomicOr(a.err, 4);
                page = min(max(page, 0), a.n_pages - 1);
            }
        });
    }
    merge_waves<T, NW>(st, lds.merge, wave, lane, [&](int c, int d, float M, float L, f32x4 A) {
        if (c >= G) return;
        if constexpr (FINISH) {
            const int n = q.slots;
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
    const int n0 = q.slots;
    const int n1 = q.bad || q.len == 0 ? 0 : (int)((q.len - q.own + a.tail_rows - 1) / a.tail_rows);
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
    extern "C" __global__ __launch_bounds__(64 * kPagedWaves) void tmac_selected_##NAME(PagedAttnArgs a) {             \
        selected_body<T, kPagedWaves>(a);                                                                              \
    }                                                                                                                  \
    extern "C" __global__ __launch_bounds__(64 * kSharedWaves) void tmac_selected_wide_##NAME(PagedAttnArgs a) {       \
        selected_body<T, kSharedWaves>(a);                                                                             \
    }                                                                                                                  \
    extern "C" __global__ __launch_bounds__(64 * kSharedWaves) void tmac_prefix_##NAME(PagedAttnArgs a) {               \
        prefix_body<T>(a);                                                                                             \
    }                                                                                                                  \
    extern "C" __global__ __launch_bounds__(64 * kPagedWaves) void tmac_tail_##NAME(PagedAttnArgs a) {                 \
        tail_body<T, kPagedWaves, false>(a);                                                                           \
    }                                                                                                                  \
    extern "C" __global__ __launch_bounds__(64 * kPagedWaves) void tmac_tail_finish_##NAME(PagedAttnArgs a) {          \
        tail_body<T, kPagedWaves, true>(a);                                                                            \
    }                                                                                                                  \
    extern "C" __global__ __launch_bounds__(64 * kSharedWaves) void tmac_tail_finish_wide_##NAME(PagedAttnArgs a) {    \
        tail_body<T, kSharedWaves, true>(a);                                                                           \
    }
TMAC_PAGED_KERNELS(f32, float)
TMAC_PAGED_KERNELS(bf16, __bf16)
TMAC_PAGED_KERNELS(f16, _Float16)
TMAC_PAGED_KERNELS(q8, q8_0_t)

extern "C" __global__ __launch_bounds__(64 * kPagedWaves) void tmac_page_scores_h4(SelectArgs a) { score_body<1>(a); }
extern "C" __global__ __launch_bounds__(64 * kPagedWaves) void tmac_page_scores_h8(SelectArgs a) { score_body<2>(a); }
extern "C" __global__ __launch_bounds__(64 * kPagedWaves) void tmac_select_short_h4(SelectArgs a) { select_short_body<1>(a); }
extern "C" __global__ __launch_bounds__(64 * kPagedWaves) void tmac_select_short_h8(SelectArgs a) { select_short_body<2>(a); }
extern "C" __global__ __launch_bounds__(256) void tmac_select_pages_256(SelectArgs a) { select_body<256>(a); }
extern "C" __global__ __launch_bounds__(1024) void tmac_select_pages_1024(SelectArgs a) { select_body<1024>(a); }
#define TMAC_MERGE_KERNELS(WPR)                                                                          \
    extern "C" __global__ __launch_bounds__(64 * kPagedWaves) void tmac_selected_merge_w##WPR(PagedAttnArgs a) { \
        selected_merge_body<WPR>(a);                                                                     \
    }                                                                                                    \
    extern "C" __global__ __launch_bounds__(64 * kPagedWaves) void tmac_shared_merge_w##WPR(PagedAttnArgs a) { \
        shared_merge_body<WPR>(a);                                                                       \
    }
TMAC_MERGE_KERNELS(1)
TMAC_MERGE_KERNELS(4)
