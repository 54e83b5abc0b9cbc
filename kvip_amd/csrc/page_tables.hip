// Page tables of a batch on the GPU: the pages, slots, positions and visibility of a step's
// tokens from the request lengths (extend), pages given back (truncate), rows of the kept tokens of
// a tree copied together (move). kvip_hip_draft.h states the rules.
//
// With need_b = ceil((len_b + count_b) / 128) - ceil(len_b / 128), request b's block j past its old ones is
// page free[top - 1 - (sum of the needs before b) - (j - old blocks)], so once the two prefix sums
// over the batch (tokens, pages) are known, every table entry and slot is independent of the others.
// What bounds it: latency (a few loads, two scans, one launch), then the 24 bytes written per token.
// Extend takes 5.5 us for 64 requests with trees of 1-9 tokens, 8.6 for 300 requests of 1-700 tokens (105000
// rows, 2.5 MB); truncate 3.9 and 4.2.
// Every workgroup does both scans itself (4 requests per thread, at most 1024) instead of a launch before
// it, counts itself on a ticket when it has read the state, and writes the entries of the requests and rows that
// it takes in turn; the last one on the ticket moves the lengths and the stack's top on. Nothing that one
// workgroup wrote is read by another in the same launch, so the ticket needs no fence.
//
// The ancestors of a tree's tokens (at most 64, one wave per request, one lane per token) come by
// pointer doubling: after round r a lane's mask holds its nearest 2^r ancestors.
#include "kvip_device.h"
#include "kvip_hip_draft.h"

namespace kvip {
namespace {

constexpr int kTableThreads = 256;
constexpr int kTableWaves = kTableThreads / 64;
constexpr int kPerThread = KVIP_DRAFT_MAX_BATCH / kTableThreads;

struct TablePlan {
    uint32_t wave_sums[kTableWaves];
    int32_t start[KVIP_DRAFT_MAX_BATCH + 1];  // first row of a request
    int32_t pages[KVIP_DRAFT_MAX_BATCH];      // pages of the requests before it
    int32_t length[KVIP_DRAFT_MAX_BATCH];     // before the step
    int32_t step[KVIP_DRAFT_MAX_BATCH];       // tokens appended / the new length
};

KVIP_DEVICE int blocks_of(int tokens) { return (tokens + kBlockTokens - 1) / kBlockTokens; }

KVIP_DEVICE int clamp_int(int x, int lo, int hi) { return min(max(x, lo), hi); }

// Counts this workgroup; true in the last one, whose turn it is to write what the others have read.
KVIP_DEVICE bool last_group(int32_t* ticket) {
    __shared__ int s_last;
    __syncthreads();  // every read of the state by this workgroup is done
    if (gridDim.x == 1) return true;
    if (threadIdx.x == 0) {
        // atomicInc wraps to 0 at the last one: ready for the next call.
        s_last = atomicInc(reinterpret_cast<uint32_t*>(ticket), gridDim.x - 1) == gridDim.x - 1;
    }
    __syncthreads();
    return s_last != 0;
}

KVIP_DEVICE uint64_t shuffle64(uint64_t v, int lane) {
    const uint32_t lo = static_cast<uint32_t>(__shfl(static_cast<int>(v), lane));
    const uint32_t hi = static_cast<uint32_t>(__shfl(static_cast<int>(v >> 32), lane));
    return static_cast<uint64_t>(hi) << 32 | lo;
}

// Page of block j of request b in the step that extend lays out.
KVIP_DEVICE int page_of(const KvipPageTableArgs& p, const TablePlan& s, int b, int j, int top) {
    const int old = blocks_of(s.length[b]);
    if (j < old) return p.block_table[static_cast<int64_t>(b) * p.max_blocks + j];
    return p.free_pages[clamp_int(top - 1 - s.pages[b] - (j - old), 0, p.num_blocks - 1)];
}

__global__ __launch_bounds__(kTableThreads) void extend_tables_kernel(const KvipPageTableArgs p) {
    __shared__ TablePlan s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int capacity = p.max_blocks * kBlockTokens;
    const int top = clamp_int(p.free_count[0], 0, p.num_blocks);
    const int most = p.parents != nullptr ? KVIP_DRAFT_MAX_NODES : p.max_tokens;
    uint32_t err = 0;

    // Rows before each request.
    int length[kPerThread], count[kPerThread];
    uint32_t rows = 0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
        const int b = tid * kPerThread + i;
        length[i] = b < p.batch ? p.lengths[b] : 0;
        count[i] = b < p.batch ? p.counts[b] : 0;
    }
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
        if (length[i] != clamp_int(length[i], 0, capacity) || count[i] < 0) err |= KVIP_STATUS_BAD_LENGTH;
        length[i] = clamp_int(length[i], 0, capacity);
        rows += min(max(count[i], 0), p.max_tokens + 1);
    }
    uint32_t total;
    uint32_t row = block_exclusive_scan(rows, s.wave_sums, &total);
    // Pages before each request, of those that can be appended.
    uint32_t pages = 0;
    int step[kPerThread];
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
        const int b = tid * kPerThread + i;
        const int n = min(max(count[i], 0), p.max_tokens + 1);
        const uint32_t end = row + n;
        const bool fits = n <= capacity - length[i] && n <= most && end <= static_cast<uint32_t>(p.max_tokens);
        if (!fits) err |= KVIP_STATUS_BAD_LENGTH;
        step[i] = fits ? n : 0;
        pages += blocks_of(length[i] + step[i]) - blocks_of(length[i]);
        if (b < p.batch) s.start[b] = static_cast<int>(min(row, static_cast<uint32_t>(p.max_tokens)));
        row = end;
    }
    uint32_t wanted, taken, given = 0;
    uint32_t page = block_exclusive_scan(pages, s.wave_sums, &wanted);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
        const int b = tid * kPerThread + i;
        const uint32_t need = blocks_of(length[i] + step[i]) - blocks_of(length[i]);
        if (need != 0 && page + need > static_cast<uint32_t>(top)) {
            err |= KVIP_STATUS_NO_PAGE;
            step[i] = 0;
        } else {
            given += need;
        }
        if (b < p.batch) {
            s.pages[b] = static_cast<int>(min(page, static_cast<uint32_t>(top)));
            s.length[b] = length[i];
            s.step[b] = step[i];
        }
        page += need;
    }
    if (tid == 0) s.start[p.batch] = static_cast<int>(min(total, static_cast<uint32_t>(p.max_tokens)));
    if (blockIdx.x == 0) report(p.status, err);
    block_exclusive_scan(given, s.wave_sums, &taken);

    if (last_group(p.ticket)) {
        for (int b = tid; b <= p.batch; b += kTableThreads) {
            p.cu_seqlens[b] = s.start[b];
            if (b == p.batch) break;
            p.lengths[b] = s.length[b] + s.step[b];
            p.bases[b] = s.length[b];
            p.steps[b] = s.step[b];
        }
        if (tid == 0) p.free_count[0] = top - static_cast<int>(taken);
    }

    // Table entries of the new pages; with a tree, also everything of its tokens: one wave per request.
    for (int b = blockIdx.x * kTableWaves + wave; b < p.batch; b += gridDim.x * kTableWaves) {
        const int begin = s.start[b], n = s.step[b], base = s.length[b];
        const int old = blocks_of(base), now = blocks_of(base + n);
        for (int j = old + lane; j < now; j += 64) {
            p.block_table[static_cast<int64_t>(b) * p.max_blocks + j] = page_of(p, s, b, j, top);
        }
        if (p.parents == nullptr) continue;
        const int there = min(s.start[b + 1] - begin, KVIP_DRAFT_MAX_NODES);  // also of a refused request
        int up = lane < there ? p.parents[begin + lane] : -1;
        if (up < -1 || up >= lane) {
            report(p.status, KVIP_STATUS_BAD_TREE);
            up = -1;
        }
        uint64_t mask = 1ull << lane;
#pragma unroll
        for (int r = 0; r < 6; ++r) {
            const uint64_t above = shuffle64(mask, max(up, 0));
            const int next = __shfl(up, max(up, 0));
            if (up >= 0) {
                mask |= above;
                up = next;
            }
        }
        if (lane < there) {
            const int at = base + lane;
            const int64_t slot = n > 0 ? static_cast<int64_t>(page_of(p, s, b, at / kBlockTokens, top)) * kBlockTokens +
                                             at % kBlockTokens : -1;
            p.visible[begin + lane] = static_cast<int64_t>(mask);
            p.positions[begin + lane] = base + __popcll(mask) - 1;
            p.slots[begin + lane] = slot;
        }
        for (int t = begin + KVIP_DRAFT_MAX_NODES + lane; t < s.start[b + 1]; t += 64) {  // a refused one's rest
            p.visible[t] = 0;
            p.positions[t] = 0;
            p.slots[t] = -1;
        }
    }
    // Rows: of every request (without parents), and behind the last one.
    const int first = p.parents == nullptr ? 0 : s.start[p.batch];
    for (int t = first + blockIdx.x * kTableThreads + tid; t < p.max_tokens; t += gridDim.x * kTableThreads) {
        int64_t slot = -1, position = 0;
        uint64_t seen = 0;
        if (t < s.start[p.batch]) {
            int lo = 0, hi = p.batch - 1;  // the last request that starts at or before t has the row
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (s.start[mid] <= t) lo = mid;
                else hi = mid - 1;
            }
            const int within = t - s.start[lo], at = s.length[lo] + within;
            position = at;
            seen = ~0ull >> (63 - min(within, 63));  // of a chain: every token up to this one
            if (within < s.step[lo]) {
                slot = static_cast<int64_t>(page_of(p, s, lo, at / kBlockTokens, top)) * kBlockTokens + at % kBlockTokens;
            }
        }
        p.slots[t] = slot;
        p.positions[t] = position;
        if (p.visible != nullptr) p.visible[t] = static_cast<int64_t>(seen);
    }
}

__global__ __launch_bounds__(kTableThreads) void truncate_tables_kernel(const KvipPageTableArgs p) {
    __shared__ TablePlan s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int capacity = p.max_blocks * kBlockTokens;
    const int top = clamp_int(p.free_count[0], 0, p.num_blocks);
    uint32_t err = 0, pages = 0;
    int length[kPerThread], target[kPerThread], base[kPerThread], step[kPerThread];
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
        const int b = tid * kPerThread + i;
        const bool in = b < p.batch;
        length[i] = in ? p.lengths[b] : 0;
        target[i] = in ? p.targets[b] : 0;
        base[i] = in && p.kept ? p.bases[b] : 0;
        step[i] = in && p.kept ? p.steps[b] : 0;
    }
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
        const int b = tid * kPerThread + i;
        if (length[i] != clamp_int(length[i], 0, capacity)) err |= KVIP_STATUS_BAD_LENGTH;
        length[i] = clamp_int(length[i], 0, capacity);
        int now = target[i];
        if (p.kept) {
            const int kept = clamp_int(now, 0, max(step[i], 0));
            if (kept != now) err |= KVIP_STATUS_BAD_LENGTH;
            now = clamp_int(base[i], 0, capacity) + min(kept, capacity);
        }
        if (now != clamp_int(now, 0, length[i])) err |= KVIP_STATUS_BAD_LENGTH;
        now = clamp_int(now, 0, length[i]);
        pages += blocks_of(length[i]) - blocks_of(now);
        if (b < p.batch) {
            s.length[b] = length[i];
            s.step[b] = now;
        }
        target[i] = now;
    }
    uint32_t freed;
    uint32_t page = block_exclusive_scan(pages, s.wave_sums, &freed);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
        const int b = tid * kPerThread + i;
        if (b < p.batch) s.pages[b] = static_cast<int>(page);
        page += blocks_of(length[i]) - blocks_of(target[i]);
    }
    const int64_t height = static_cast<int64_t>(top) + freed;
    if (height > p.num_blocks) err |= KVIP_STATUS_BAD_BLOCK;  // pages that are in the stack already
    if (blockIdx.x == 0) report(p.status, err);
    if (last_group(p.ticket)) {
        for (int b = tid; b < p.batch; b += kTableThreads) {
            p.lengths[b] = p.bases[b] = s.step[b];
            p.steps[b] = 0;
        }
        if (tid == 0) p.free_count[0] = static_cast<int>(min(height, static_cast<int64_t>(p.num_blocks)));
    }
    for (int b = blockIdx.x * kTableWaves + wave; b < p.batch; b += gridDim.x * kTableWaves) {
        const int first = blocks_of(s.step[b]);
        int32_t* table = p.block_table + static_cast<int64_t>(b) * p.max_blocks;
        for (int j = first + lane; j < blocks_of(s.length[b]); j += 64) {
            const int64_t at = height - 1 - s.pages[b] - (j - first);
            if (at >= 0 && at < p.num_blocks) p.free_pages[at] = table[j];
            table[j] = -1;
        }
    }
}

// One workgroup per (request, cache). A thread takes the same 4 bytes of every row, so the rows that it
// still has to read are never ones that it has written: rows are read 8 at a time, and the row at
// place i comes from a place >= i. A path is looked up 64 places at a time.
constexpr int kMoveAhead = 8;
constexpr int kMovePlaces = 64;
__global__ __launch_bounds__(256) void move_rows_kernel(const KvipPageTableArgs p) {
    __shared__ int64_t s_from[kMovePlaces], s_to[kMovePlaces];  // slots
    __shared__ int s_count;
    const int b = blockIdx.x, tid = threadIdx.x;
    const int capacity = p.max_blocks * kBlockTokens;
    const int base = clamp_int(p.bases[b], 0, capacity);
    const int step = min(p.steps[b], capacity - base);
    const int kept = clamp_int(p.targets[b], 0, max(step, 0));
    const int want = min(kept, p.path_stride);
    if (tid == 0 && blockIdx.y == 0 && want < kept) report(p.status, KVIP_STATUS_BAD_LENGTH);
    const int32_t* table = p.block_table + static_cast<int64_t>(b) * p.max_blocks;
    const int32_t* path = p.path + static_cast<int64_t>(b) * p.path_stride;
    const KvipPagedRows c = p.rows[blockIdx.y];
    auto at = [&](int64_t slot) {
        return reinterpret_cast<uint32_t*>(c.base + slot / kBlockTokens * c.block_stride + slot % kBlockTokens * c.row_stride);
    };
    for (int first = 0; first < want; first += kMovePlaces) {
        if (tid < kMovePlaces) {
            const int place = first + tid;
            const bool named = place < want;
            const int node = named ? path[place] : -1;
            const int before = named && place > 0 ? path[place - 1] : -1;
            bool ok = named && node >= 0 && node < step && node > before;
            int64_t from = 0, to = 0;
            uint32_t err = named && !ok ? KVIP_STATUS_BAD_TREE : 0u;
            if (ok) {
                const int src = base + node, dst = base + place;
                const int src_page = table[src / kBlockTokens], dst_page = table[dst / kBlockTokens];
                ok = static_cast<unsigned>(src_page) < static_cast<unsigned>(p.num_blocks) &&
                     static_cast<unsigned>(dst_page) < static_cast<unsigned>(p.num_blocks);
                if (!ok) err = KVIP_STATUS_BAD_BLOCK;
                from = static_cast<int64_t>(src_page) * kBlockTokens + src % kBlockTokens;
                to = static_cast<int64_t>(dst_page) * kBlockTokens + dst % kBlockTokens;
            }
            s_from[tid] = from;
            s_to[tid] = to;
            const unsigned long long bad = __ballot(named && !ok);
            // The rows before the first bad one.
            if (tid == 0) s_count = bad != 0 ? __ffsll(bad) - 1 : min(want - first, kMovePlaces);
            if (blockIdx.y == 0) report(p.status, err);
        }
        __syncthreads();
        const int count = s_count;
        for (int64_t w = tid; w < c.row_bytes / 4; w += 256) {
            for (int i = 0; i < count; i += kMoveAhead) {
                uint32_t v[kMoveAhead];
#pragma unroll
                for (int k = 0; k < kMoveAhead; ++k) {
                    if (i + k < count) v[k] = at(s_from[i + k])[w];
                }
#pragma unroll
                for (int k = 0; k < kMoveAhead; ++k) {
                    if (i + k < count) at(s_to[i + k])[w] = v[k];
                }
            }
        }
        if (count < kMovePlaces) break;  // uniform: the path's end, or a bad place
        __syncthreads();
    }
}

bool valid_tables(const KvipPageTableArgs* a) {
    return a != nullptr && a->block_table && a->lengths && a->free_pages && a->free_count && a->bases && a->steps &&
           a->ticket && a->batch >= 1 && a->batch <= KVIP_DRAFT_MAX_BATCH && a->max_blocks >= 1 &&
           a->max_blocks <= (1 << 24) / kBlockTokens && a->num_blocks >= 1 && a->num_blocks < (1 << 24);
}

int table_groups(int batch, int tokens) {
    // 512 rows each: 105000 rows take 12.5 us with truncate (1024: 13.3, 256: 13.7, for the tickets).
    const int by_request = (batch + kTableWaves - 1) / kTableWaves, by_row = (tokens + 511) / 512;
    return by_request > by_row ? by_request : by_row;
}

}  // namespace
}  // namespace kvip

extern "C" uint32_t kvip_hip_draft_abi_version(void) { return KVIP_DRAFT_ABI_VERSION; }

extern "C" uint32_t kvip_hip_page_tables_extend(const KvipPageTableArgs* a, void* stream) {
    const bool ok = kvip::valid_tables(a) && a->counts && a->cu_seqlens && a->positions && a->slots &&
                    (a->parents == nullptr || a->visible != nullptr) && a->max_tokens >= 1 &&
                    a->max_tokens <= KVIP_DRAFT_MAX_TOKENS;
    if (!ok) return KVIP_ERR_INVALID;
    hipLaunchKernelGGL(kvip::extend_tables_kernel, dim3(kvip::table_groups(a->batch, a->max_tokens)),
                       dim3(kvip::kTableThreads), 0, static_cast<hipStream_t>(stream), *a);
    return static_cast<uint32_t>(hipGetLastError());
}

extern "C" uint32_t kvip_hip_page_tables_move(const KvipPageTableArgs* a, void* stream) {
    const bool ok = kvip::valid_tables(a) && a->targets && a->path && a->path_stride >= 1 && a->row_sets >= 0 &&
                    a->row_sets <= 65535 && (a->row_sets == 0 || a->rows);
    if (!ok) return KVIP_ERR_INVALID;
    if (a->row_sets == 0) return KVIP_OK;
    hipLaunchKernelGGL(kvip::move_rows_kernel, dim3(a->batch, a->row_sets), dim3(256), 0,
                       static_cast<hipStream_t>(stream), *a);
    return static_cast<uint32_t>(hipGetLastError());
}

extern "C" uint32_t kvip_hip_page_tables_truncate(const KvipPageTableArgs* a, void* stream) {
    if (!kvip::valid_tables(a) || a->targets == nullptr) return KVIP_ERR_INVALID;
    hipLaunchKernelGGL(kvip::truncate_tables_kernel, dim3(kvip::table_groups(a->batch, 0)), dim3(kvip::kTableThreads), 0,
                       static_cast<hipStream_t>(stream), *a);
    return static_cast<uint32_t>(hipGetLastError());
}
