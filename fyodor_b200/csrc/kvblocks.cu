// kvblocks.cu - block tables and slot maps of a paged KV cache, built on the
// device from request lengths.
//
// need[r] = ceil((len + new) / block) - ceil(len / block) blocks per request;
// the exclusive prefix sums of need and of the row counts say which free
// blocks and which rows are a request's. The step is a few KB of integers:
// bound by latency, so it is one launch. Every CTA scans all requests (two
// values each, in shared memory) and then writes its share of the requests,
// rows and new table entries, so no CTA waits for another.
#include "common.cuh"
#include "kernels.h"
#include "fyodor_b200.h"

namespace fyb {

constexpr unsigned KB_THREADS = 512, KB_REQUESTS = 16384;

struct KvBlocksArgs {
    const int *lengths, *new_tokens, *free_list, *free_count;
    int *table, *lengths_out, *free_count_out, *row_start, *slots, *positions, *row_request, *status;
    size_t stride;
    unsigned n, shift, max_rows;
};

// Inclusive scan over the CTA of (a, b), sums held at most at (la, lb): the
// saturating sum is associative, so the scan is exact below the limits.
FYB_DEV uint2 kb_scan(uint2 v, unsigned la, unsigned lb, uint2 *warp_sums)
{
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (unsigned o = 1; o < 32; o <<= 1) {
        const unsigned a = __shfl_up_sync(0xffffffffu, v.x, o), b = __shfl_up_sync(0xffffffffu, v.y, o);
        if (lane >= o) v = make_uint2(min(v.x + a, la), min(v.y + b, lb));
    }
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    for (unsigned w = 0; w < warp; ++w) v = make_uint2(min(v.x + warp_sums[w].x, la), min(v.y + warp_sums[w].y, lb));
    return v;
}

// The last r with from[r] <= x; from[0] = 0 <= x.
FYB_DEV unsigned kb_owner(const unsigned *from, unsigned n, unsigned x)
{
    unsigned lo = 0, hi = n;  // from[lo] <= x, and x < from[hi] or hi == n
    while (hi - lo > 1) {
        const unsigned mid = (lo + hi) / 2;
        if (from[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(KB_THREADS) kv_blocks_kernel(KvBlocksArgs A)
{
    extern __shared__ unsigned kb_smem[];
    unsigned *row = kb_smem, *blk = kb_smem + A.n + 1;  // exclusive prefix sums [n + 1]
    __shared__ uint2 warp_sums[KB_THREADS / 32];
    const unsigned size = 1u << A.shift, tid = threadIdx.x, n = A.n;
    const unsigned count = (unsigned)max(A.free_count[0], 0);
    const unsigned row_limit = A.max_rows + 1, blk_limit = count + 1;
    const long long holds = min((long long)A.stride << A.shift, 0x7fffffffll);  // lengths and positions are 31 bits
    auto valid = [&](int len, int more) { return len >= 0 && more >= 0 && (long long)len + more <= holds; };
    auto blocks = [&](int tokens) { return (unsigned)(((long long)tokens + size - 1) >> A.shift); };

    unsigned row_carry = 0, blk_carry = 0;
    if (tid == 0) row[0] = blk[0] = 0;
    for (unsigned base = 0; base < n; base += KB_THREADS) {
        const unsigned r = base + tid;
        const int len = r < n ? A.lengths[r] : 0, more = r < n ? A.new_tokens[r] : 0;
        const bool ok = valid(len, more);
        uint2 v = make_uint2(ok ? min((unsigned)more, row_limit) : 0u, 0u);
        // rows first: a request that ends beyond max_rows needs no blocks
        uint2 t = kb_scan(v, row_limit, 1u, warp_sums);
        t.x = min(t.x + row_carry, row_limit);
        __syncthreads();
        if (ok && t.x <= A.max_rows) v.y = min(blocks(len + more) - blocks(len), blk_limit);
        v.x = 0;
        uint2 u = kb_scan(v, 1u, blk_limit, warp_sums);
        u.y = min(u.y + blk_carry, blk_limit);
        if (r < n) { row[r + 1] = t.x; blk[r + 1] = u.y; }
        __syncthreads();
        row_carry = row[min(base + KB_THREADS, n)];
        blk_carry = blk[min(base + KB_THREADS, n)];
    }
    const unsigned first = blockIdx.x * KB_THREADS + tid, step = gridDim.x * KB_THREADS;
    // 0 served, 1 too few blocks, 2 invalid
    auto state = [&](unsigned r, int len, int more) {
        if (!valid(len, more) || row[r + 1] > A.max_rows) return 2;
        return blocks(len + more) == blocks(len) || blk[r + 1] <= count ? 0 : 1;
    };
    for (unsigned r = first; r < n; r += step) {
        const int len = A.lengths[r], more = A.new_tokens[r], st = state(r, len, more);
        A.status[r] = st;
        A.lengths_out[r] = st == 0 ? len + more : len;
        A.row_start[r + 1] = (int)min(row[r + 1], A.max_rows);
    }
    // requests are refused from the first whose blocks run out, so the blocks
    // taken are the longest prefix that fits
    unsigned taken = blk[kb_owner(blk, n + 1, count)];
    if (first == 0) {
        A.row_start[0] = 0;
        A.free_count_out[0] = (int)(count - taken);
    }
    for (unsigned j = first; j < taken; j += step) {
        const unsigned r = kb_owner(blk, n, j);
        A.table[(size_t)r * A.stride + blocks(A.lengths[r]) + (j - blk[r])] = A.free_list[count - 1 - j];
    }
    const unsigned total = min(row[n], A.max_rows);
    for (unsigned i = first; i < A.max_rows; i += step) {
        int slot = -1, pos = 0, who = -1;
        if (i < total) {
            const unsigned r = kb_owner(row, n, i);
            const int len = A.lengths[r], more = A.new_tokens[r];
            who = (int)r;
            pos = len + (int)(i - row[r]);
            if (state(r, len, more) == 0) {
                const unsigned b = (unsigned)pos >> A.shift, old = blocks(len);
                const int id = b < old ? A.table[(size_t)r * A.stride + b] : A.free_list[count - 1 - (blk[r] + b - old)];
                slot = id * (int)size + (int)((unsigned)pos & (size - 1));
            }
        }
        A.slots[i] = slot;
        A.positions[i] = pos;
        A.row_request[i] = who;
    }
}

__global__ void __launch_bounds__(KB_THREADS) kv_release_kernel(int *lengths, const int *keep, unsigned n, int *table,
    size_t stride, unsigned shift, int *free_list, int *free_count, unsigned capacity)
{
    __shared__ uint2 warp_sums[KB_THREADS / 32];
    __shared__ unsigned carry_s;
    const unsigned size = 1u << shift, tid = threadIdx.x, limit = 1u << 30;
    unsigned carry = (unsigned)max(free_count[0], 0);
    auto blocks = [&](int tokens) { return (long long)((unsigned)tokens + size - 1) >> shift; };
    for (unsigned base = 0; base < n; base += KB_THREADS) {
        const unsigned r = base + tid;
        const int len = r < n ? max(lengths[r], 0) : 0, left = r < n ? min(max(keep[r], 0), len) : 0;
        const long long held = blocks(len), stay = blocks(left);
        const unsigned mine = held <= (long long)stride ? (unsigned)(held - stay) : 0u;
        const uint2 v = kb_scan(make_uint2(mine, 0u), limit, 1u, warp_sums);
        const unsigned end = min(v.x + carry, limit);
        // what would not fit stays with its request, and so does all after it
        const bool fits = end <= capacity || carry + v.x == carry;
        if (fits && left < len) {
            for (unsigned b = 0; b < mine; ++b) {
                int *entry = table + (size_t)r * stride + (size_t)stay + b;
                free_list[end - mine + b] = *entry;
                *entry = -1;
            }
            lengths[r] = left;
        }
        if (tid == 0) carry_s = carry;
        __syncthreads();
        if (fits && mine) atomicMax(&carry_s, end);
        const bool full = __syncthreads_or(!fits);
        carry = carry_s;
        __syncthreads();
        if (full) break;
    }
    if (tid == 0) free_count[0] = (int)carry;
}

static int log2_block(unsigned size)
{
    for (int s = 0; s < 20; ++s) if (size == 1u << s) return s;
    return -1;
}

}  // namespace fyb

using namespace fyb;

extern "C" int fyb_kv_blocks(const int32_t *lengths, const int32_t *new_tokens, uint32_t requests, int32_t *table,
    size_t stride, uint32_t block_size, const int32_t *free_list, const int32_t *free_count, int32_t *lengths_out,
    int32_t *free_count_out, int32_t *row_start, int32_t *slots, int32_t *positions, int32_t *row_request,
    uint32_t max_rows, int32_t *status, void *stream)
{
    const int shift = log2_block(block_size);
    if (!lengths || !new_tokens || !table || !free_list || !free_count || !lengths_out || !free_count_out ||
        !row_start || !status || (max_rows && (!slots || !positions || !row_request)) || requests == 0 ||
        requests > KB_REQUESTS || shift < 0 || stride == 0 || stride > 0x7fffffffu || max_rows >= 1u << 30 ||
        lengths_out == lengths || free_count_out == free_count)
        return -1;
    const KvBlocksArgs A{lengths, new_tokens, free_list, free_count, table, lengths_out, free_count_out, row_start,
                         slots, positions, row_request, status, stride, requests, (unsigned)shift, max_rows};
    const size_t smem = (size_t)2 * (requests + 1) * sizeof(unsigned);
    static std::atomic<unsigned> allowed{0};
    if (smem > 48 * 1024 && allow_shared((const void *)kv_blocks_kernel, 2 * (KB_REQUESTS + 1) * sizeof(unsigned), allowed))
        return -2;
    const size_t most = std::max<size_t>(max_rows, requests);
    const unsigned grid = (unsigned)std::min<size_t>((most + KB_THREADS - 1) / KB_THREADS, 148);
    kv_blocks_kernel<<<grid, KB_THREADS, smem, (cudaStream_t)stream>>>(A);
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

extern "C" int fyb_kv_release(int32_t *lengths, const int32_t *keep, uint32_t requests, int32_t *table, size_t stride,
    uint32_t block_size, int32_t *free_list, int32_t *free_count, uint32_t free_capacity, void *stream)
{
    const int shift = log2_block(block_size);
    if (!lengths || !keep || !table || !free_list || !free_count || requests == 0 || requests > KB_REQUESTS ||
        shift < 0 || stride == 0 || stride > 0x7fffffffu || free_capacity >= 1u << 30)
        return -1;
    kv_release_kernel<<<1, KB_THREADS, 0, (cudaStream_t)stream>>>(lengths, keep, requests, table, stride,
                                                                  (unsigned)shift, free_list, free_count, free_capacity);
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
}
