// w4a8_pages.cu -- the pages of a paged cache kept on the device: a step's page table,
// lengths, offsets, slots and rotary positions made from the tokens that each sequence
// brings, pages taken from a stack of free ones, and given back.
//
// A sequence of len tokens holds ceil(len / S) pages.  A plan over sequences 0 .. B - 1, bringing n_i tokens each:
//
//   need_i = ceil((len_i + n_i) / S) - ceil(len_i / S)          pages off the stack's top, in the sequences' order
//   cu_i   = n_0 + .. + n_{i - 1}                               (prefix sums, as are the pages')
//   slot   = page(pos / S) S + pos % S                          of a token at position pos = len_i + its number
//
// Shrinking is its inverse, page by page: sequences from the last to the first, each one's pages
// from the last to the first, onto the stack.
//
// Rotary positions on three axes: a grid of t x h x w tokens whose first token is number
// `start` of its sequence begins at that token's text position o and counts (o + r / (h w), o + r / w % h, o + r % w);
// what follows goes on at o + max(t, h, w).
//
// One launch.  Every block finds all sums itself (up to 2048 sequences: eight or two a thread, a scan over the block), so no
// block waits for another, and does its share of table rows and tokens.  The lengths and the stack's height, which all blocks
// read first, are set by the block that finishes last.  A step that cannot be (a row twice or outside, too few pages, ...)
// changes nothing: its tables say "no page" and "no tokens", and the status word says why.
#include <algorithm>

#include "w4a8_common.cuh"
#include "w4a8_kernels.h"

namespace w4a8 {

namespace {

constexpr int kSmall = 256, kLarge = 1024;                     // threads of a block

struct Sums {
    int64_t tokens, pages;
};

__device__ __forceinline__ Sums add(Sums a, Sums b) { return {a.tokens + b.tokens, a.pages + b.pages}; }

__device__ __forceinline__ Sums shfl_up(Sums v, int o)
{
    return {static_cast<int64_t>(__shfl_up_sync(0xffffffffu, v.tokens, o)), static_cast<int64_t>(__shfl_up_sync(0xffffffffu, v.pages, o))};
}

// What a block knows about the whole step: offsets of each sequence's tokens and pages, its row and length.
struct Step {
    int cu[kMaxPlanBatch + 1];
    int pages[kMaxPlanBatch + 1];
    int row[kMaxPlanBatch];
    int len[kMaxPlanBatch];
    uint32_t seen[kMaxPlanRows / 32];
    Sums warp_sums[kLarge / 32];
    int bad, last;
};

__device__ __forceinline__ int pages_of(int64_t len, int log2) { return static_cast<int>((len + (int64_t(1) << log2) - 1) >> log2); }

// Fills `st`; 0, or why the step cannot be.  SHRINK: counts are the lengths to keep (null: 0), pages those given back.
template <int T, bool SHRINK>
__device__ int gather(const PagesParams& p, Step& st, int& height)
{
    constexpr int PER = kMaxPlanBatch / T, WARPS = T / 32;
    const int tid = threadIdx.x, B = p.batch, per = (B + T - 1) / T;
    int row[PER], count[PER], len[PER], need[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int i = tid * per + j;
        const bool on = j < per && i < B;
        row[j] = on ? p.rows[i] : -1;
        count[j] = on && p.counts ? p.counts[i] : 0;
    }
    for (int i = tid; i < (p.sequences + 31) / 32; i += T) st.seen[i] = 0;
    if (tid == 0) st.bad = 0;
    height = *p.free_count;
#pragma unroll
    for (int j = 0; j < PER; ++j) len[j] = row[j] >= 0 && row[j] < p.sequences ? p.lens[row[j]] : 0;
    __syncthreads();
    int bad = height < 0 || height > p.pages ? kPlanState : 0;
    Sums mine{0, 0};
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int i = tid * per + j, n = count[j];
        need[j] = 0;
        if (j >= per || i >= B) continue;
        const int held = pages_of(len[j], p.page_log2);
        if (row[j] < 0 || row[j] >= p.sequences || (atomicOr(&st.seen[row[j] >> 5], 1u << (row[j] & 31)) >> (row[j] & 31) & 1u)) {
            bad |= kPlanRow;
        } else if (len[j] < 0 || held > p.columns) {
            bad |= kPlanState;
        } else if (SHRINK) {
            if (n < 0 || n > len[j]) bad |= kPlanCount;
            else need[j] = held - pages_of(n, p.page_log2);
        } else if (n < 0 || n > p.tokens) {
            bad |= n < 0 ? kPlanCount : kPlanTokens;
        } else if (const int all = pages_of(static_cast<int64_t>(len[j]) + n, p.page_log2); all > p.columns) {
            bad |= kPlanColumns;
        } else {
            need[j] = all - held;
        }
        st.row[i] = row[j];
        st.len[i] = len[j];
        mine = add(mine, {SHRINK ? 0 : n, need[j]});
    }
    Sums x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const Sums y = shfl_up(x, o);
        if (static_cast<int>(lane_id()) >= o) x = add(x, y);
    }
    if (lane_id() == 31) st.warp_sums[warp_id()] = x;
    if (bad) atomicOr(&st.bad, bad);
    __syncthreads();
    Sums at{x.tokens - mine.tokens, x.pages - mine.pages}, total{0, 0};
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        if (w < static_cast<int>(warp_id())) at = add(at, st.warp_sums[w]);
        total = add(total, st.warp_sums[w]);
    }
    bad = st.bad;
    if (bad) return bad;                                      // (the sums are those of the others)
    if (!SHRINK && total.tokens > p.tokens) bad |= kPlanTokens;
    if (SHRINK ? height + total.pages > p.pages : total.pages > height) bad |= SHRINK ? kPlanState : kPlanPages;
    if (bad) return bad;                                      // (sums past here fit 32 bits)
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int i = tid * per + j;
        if (j >= per || i >= B) continue;
        st.cu[i] = static_cast<int>(SHRINK ? count[j] : at.tokens);      // SHRINK: the length to keep
        st.pages[i] = static_cast<int>(at.pages);
        at = add(at, {SHRINK ? 0 : count[j], need[j]});
    }
    if (tid == 0) {
        st.cu[B] = static_cast<int>(total.tokens);
        st.pages[B] = static_cast<int>(total.pages);
    }
    __syncthreads();
    return 0;
}

// Whether this block is the last to come here; all others have read what it now may set.
__device__ __forceinline__ bool last_block(const PagesParams& p, Step& st)
{
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        st.last = atomicAdd(p.ticket, 1u) == gridDim.x - 1;
        if (st.last) *p.ticket = 0;
    }
    __syncthreads();
    return st.last != 0;
}

// The position on each axis of token `pos` of a sequence with grids [g0, g1).
__device__ __forceinline__ void place(const PagesParams& p, int g0, int g1, int pos, int64_t (&out)[3])
{
    int64_t shift = 0;                                        // text position minus token number, past the grids so far
    for (int g = g0; g < g1; ++g) {
        const int4 s = reinterpret_cast<const int4*>(p.segs)[g];
        if (s.x > pos) break;
        if (s.y <= 0 || s.z <= 0 || s.w <= 0) continue;       // holds no tokens
        const int64_t hw = static_cast<int64_t>(s.z) * s.w, r = static_cast<int64_t>(pos) - s.x;
        if (r / s.y < hw) {                                   // r < t h w, which may pass 64 bits
            const int64_t o = s.x + shift;
            out[0] = o + r / hw;
            out[1] = o + r / s.w % s.z;
            out[2] = o + r % s.w;
            return;
        }
        shift += max(s.y, max(s.z, s.w)) - hw * s.y;
    }
    out[0] = out[1] = out[2] = pos + shift;
}

template <int T>
__global__ void __launch_bounds__(T) pages_plan_kernel(const PagesParams p)
{
    __shared__ Step st;
    pdl_wait();
    int height;
    const int bad = gather<T, false>(p, st, height), B = p.batch;
    const int tid = blockIdx.x * T + threadIdx.x, all = gridDim.x * T, S = 1 << p.page_log2;

    for (int i = tid; i <= B; i += all) {
        p.cu[i] = bad ? 0 : st.cu[i];
        if (i < B) p.kv_lens[i] = bad ? 0 : st.len[i] + st.cu[i + 1] - st.cu[i];
    }
    // Table rows, 512 columns a warp at a time: the pages held, the new ones, none.  Four columns an access where
    // rows suit that.
    const bool vec = p.columns % 4 == 0 && (reinterpret_cast<uintptr_t>(p.table) | reinterpret_cast<uintptr_t>(p.page_table)) % 16 == 0;
    const int span = vec ? 512 : 128, chunks = (p.columns + span - 1) / span;
    for (int64_t c = tid >> 5; c < static_cast<int64_t>(B) * chunks; c += all >> 5) {
        const int i = static_cast<int>(c / chunks), c0 = static_cast<int>(c - static_cast<int64_t>(i) * chunks) * span;
        int before = 0, after = 0, row = 0, taken = 0;
        if (!bad) {
            row = st.row[i];
            taken = st.pages[i];
            before = pages_of(st.len[i], p.page_log2);
            after = before + st.pages[i + 1] - taken;
        }
        int32_t* held = p.table + static_cast<int64_t>(row) * p.columns;
        int32_t* out = p.page_table + static_cast<int64_t>(i) * p.columns;
        const auto fresh = [&](int col) {                     // a new page, or none
            if (col >= after) return -1;
            const int id = p.free[height - 1 - (taken + col - before)];
            held[col] = id;
            return id;
        };
        if (vec) {
            int4 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int col = c0 + k * 128 + static_cast<int>(lane_id()) * 4;
                v[k] = make_int4(-1, -1, -1, -1);
                if (col < before) v[k] = *reinterpret_cast<const int4*>(held + col);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int col = c0 + k * 128 + static_cast<int>(lane_id()) * 4;
                if (col >= p.columns) break;
                if (col + 4 > before) {                       // (what a row holds past its pages is no page)
                    v[k].x = col < before ? v[k].x : fresh(col);
                    v[k].y = col + 1 < before ? v[k].y : fresh(col + 1);
                    v[k].z = col + 2 < before ? v[k].z : fresh(col + 2);
                    v[k].w = fresh(col + 3);
                }
                *reinterpret_cast<int4*>(out + col) = v[k];
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int col = c0 + k * 32 + lane_id();
                if (col >= p.columns) break;
                out[col] = col < before ? held[col] : fresh(col);
            }
        }
    }
    if (p.slots || p.positions) {
        const int total = bad ? 0 : st.cu[B];
        for (int64_t t = tid; t < p.tokens; t += all) {
            int slot = -1;
            int64_t at[3] = {0, 0, 0};
            if (t < total) {
                int lo = 0, hi = B;                           // the last i with cu[i] <= t (it has tokens)
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (st.cu[mid] <= t) lo = mid;
                    else hi = mid;
                }
                const int i = lo, pos = st.len[i] + static_cast<int>(t - st.cu[i]);
                if (p.slots) {
                    const int col = pos >> p.page_log2, before = pages_of(st.len[i], p.page_log2);
                    const int id = col < before ? p.table[static_cast<int64_t>(st.row[i]) * p.columns + col]
                                                : p.free[height - 1 - (st.pages[i] + col - before)];
                    slot = (id << p.page_log2) + (pos & (S - 1));
                }
                if (p.segs) {
                    const int g0 = min(max(p.seg_cu[i], 0), p.n_segs), g1 = min(max(p.seg_cu[i + 1], 0), p.n_segs);
                    place(p, g0, g1, pos, at);
                } else {
                    at[0] = at[1] = at[2] = pos;
                }
            }
            if (p.slots) p.slots[t] = slot;
            if (p.positions)
                for (int a = 0; a < p.axes; ++a) p.positions[a * p.tokens + t] = static_cast<int32_t>(at[min(a, 2)]);
        }
    }
    if (!last_block(p, st)) return;
    if (bad) {
        if (threadIdx.x == 0) atomicCAS(p.status, 0, bad);
        return;
    }
    for (int i = threadIdx.x; i < B; i += T) p.lens[st.row[i]] = st.len[i] + st.cu[i + 1] - st.cu[i];
    if (threadIdx.x == 0) *p.free_count = height - st.pages[B];
}

template <int T>
__global__ void __launch_bounds__(T) pages_shrink_kernel(const PagesParams p)
{
    __shared__ Step st;
    pdl_wait();
    int height;
    const int bad = gather<T, true>(p, st, height), B = p.batch;
    const int tid = blockIdx.x * T + threadIdx.x, all = gridDim.x * T;
    if (!bad)
        for (int i = tid >> 5; i < B; i += all >> 5) {
            const int held = pages_of(st.len[i], p.page_log2), n = st.pages[i + 1] - st.pages[i];
            int32_t* row = p.table + static_cast<int64_t>(st.row[i]) * p.columns;
            const int base = height + st.pages[B] - st.pages[i + 1];      // the later sequences' pages lie below
            for (int k = lane_id(); k < n; k += 32) {
                p.free[base + k] = row[held - 1 - k];
                row[held - 1 - k] = -1;
            }
        }
    if (!last_block(p, st)) return;
    if (bad) {
        if (threadIdx.x == 0) atomicCAS(p.status, 0, bad);
        return;
    }
    for (int i = threadIdx.x; i < B; i += T) p.lens[st.row[i]] = st.cu[i];
    if (threadIdx.x == 0) *p.free_count = height + st.pages[B];
}

// Blocks of 1024 threads for large batches, whose sums take a block of 256 several rounds (2048 sequences of 1024
// columns: plan 20 us by 256, 9.5 by 1024), of 256 for the others (1,000 of 512: 6.6 and 9.4), as many as there is work
// for: two of `pieces` to a warp.
template <typename Kern>
cudaError_t launch(Kern small, Kern large, const PagesParams& p, int64_t pieces, cudaStream_t stream)
{
    const bool many = p.batch > 4 * kSmall;
    const int threads = many ? kLarge : kSmall;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(148, pieces * 16 / threads))));
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, many ? large : small, p);
}

}  // namespace

cudaError_t launch_pages_plan(const PagesParams& p, cudaStream_t stream)
{
    const int span = p.columns % 4 == 0 ? 512 : 128;
    const int64_t rows = static_cast<int64_t>(p.batch) * ((p.columns + span - 1) / span);
    // A warp for each row's span (plan and shrink: 256 rows of 512 columns 9.5 us so, 10.4 by half the warps; 2048 of 1024
    // 15.6 and 17.1; 1,162 of 13 columns 12.9 and 13.5, by the columns alone 16.8), a piece for eight tokens: finding one
    // among grids is a chain (12 prompts of 2,000 with four grids each 11.5 us so, 14.3 by a quarter of the blocks).
    return launch(pages_plan_kernel<kSmall>, pages_plan_kernel<kLarge>, p, std::max(2 * rows, (p.tokens + 7) / 8), stream);
}

cudaError_t launch_pages_shrink(const PagesParams& p, cudaStream_t stream)
{
    return launch(pages_shrink_kernel<kSmall>, pages_shrink_kernel<kLarge>, p, p.batch, stream);
}

}  // namespace w4a8
