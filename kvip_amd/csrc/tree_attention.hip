// Attention of a request's step tokens (a tree of drafted tokens) over its paged KV rows; the rules
// stand in kvip_hip_draft.h. A row of the cache holds 512 fp8 e4m3 features with one fp32 scale per 128
// and 64 bf16 rotary features: key = [nope * scale, rope], value = nope * scale.
//
// The rows of the problem are a request's (step token, head) pairs, which all read the same cache rows.
// A workgroup of 4 waves takes R groups of 32 rows (R = 2, 4) by 4 / R streams of 32-token tiles, a wave per
// group and stream. A wave keeps its 32 queries (128 registers) and its 32 x 512 accumulator (the 256
// accumulation registers; one wave per SIMD has 512 in all) and exchanges nothing until the streams are
// merged at the end:
//   - A tile stays as it is in the cache: direct-to-LDS loads put its fp8 bytes into a ring of three slots.
//   - Logits are computed transposed (tokens x rows): bf16 MFMA of the key bytes, converted as they are read
//     (exact), with the query; a scale group's dot products are summed on their own and added as
//     fma(group, scale, s) in fp32.
//   - So a lane holds one row's logits of 16 tokens: the softmax takes one lane swap per tile, and the
//     probabilities times the group's scale (rounded once to bf16) are the value product's operand in the
//     lane that has them, as the order of tokens along K is free (they wait in LDS, in 32 bits, while the
//     next tile's logits need the registers). The value operand (8 tokens of one feature per lane)
//     comes from the token-major tile by transposing LDS reads.
//   - The running maximum is raised lazily, when a tile exceeds it by kTaMargin.
//   - One wave per SIMD hides nothing by itself, so the tile loop is one stretch of 68 MFMAs with everything
//     else in between: the logits of tile t + 1, then the values of tile t with the softmax of tile t + 1
//     beside them; operands are read from LDS several products ahead and converted one ahead.
//
// The (request, row tile, token steps) are laid out in one line and cut into shares, one per workgroup, so
// that ragged batches keep every CU busy; what a share has of an item that others share goes to the
// workspace, and a second launch joins the parts.
//
// What bounds it. Many rows per cache row (8 requests x 12 tokens x 128 heads on 2000-8192 rows: 190 us, 795
// TFLOP/s, 125 us at the rate of a large bf16 product): the instructions between the MFMAs, 10 VALU and 1.4 LDS ones
// per MFMA, 4 of them conversions that each of the four waves does for itself (MFMA busy 38 % of the
// cycles, waiting 18 %), at the 2.2 to 2.4 GHz that the card holds under this load. Few rows (64
// requests x 4 tokens x 16 heads on 1000-16384 rows: 126 us, 2.97 TB/s): the same loop at 2.0 GHz beside the
// loads. Short contexts: a chain of latencies (lengths, page, tile and queries, two steps, join).
// Dropped after measuring: two waves per SIMD that split the features (310 us for the first of these,
// which then took 224), the query as two fp8 terms against the key's bytes (261), touching the next
// tile's lines a step ahead (+3 %), queries through LDS (+5 %).
#include <type_traits>

#include "kvip_hip_draft.h"
#include "lds_async.h"

namespace kvip {
namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) const f32x4* LdsF32x4;
typedef __attribute__((address_space(3))) f32x4* LdsF32x4Out;
typedef __attribute__((address_space(3))) i32x2* LdsI32x2;

constexpr int kTaThreads = 256;
constexpr int kTaWaves = 4;
constexpr int kTaRows = 32;                 // rows per wave (MFMA N)
constexpr int kTaTile = 32;                 // tokens per tile
constexpr int kTaSlots = 3;                 // tiles of a stream's ring
constexpr int kKeyDim = 576;                // 512 nope + 64 rope
constexpr int kValueDim = 512;
constexpr int kScaleGroups = 4;
constexpr int kBlocks = kValueDim / 32;     // accumulator blocks of 32 features
constexpr int kTaGroups = 256;              // shares: one workgroup per CU
constexpr int kMinSteps = 2;                // steps of a share, at least: 900 cache rows take 20.8 us (1: 22.6, 3: 22.4, 4: 23.3)
// What an item's start costs, in steps (the queries' loads, the first tile's). 200 requests of 4 tokens x 16 heads on
// 100-1500 rows take 67.5 us (3: 73.9, 4: 71.3, 8: 71.0), 40 of 8 tokens x 128 heads on 100-600 rows 94.6 (109, 98, 95);
// long contexts move by 1 %.
constexpr int kHeadSteps = 6;
// Waves of the join, at most, where items allow. 80 requests of 4 tokens x 16 heads on 2000-8000 rows take 101.7 us
// (4096: 104.0, 16384: 103.8); most other batches move by 1 %.
constexpr int kJoinWaves = 8192;
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f;
constexpr float kTaMargin = 8.0f * kLog2e;

constexpr int kNopeSlot = kTaTile * kValueDim;
constexpr int kRopeSlot = kTaTile * 128;
constexpr int kScaleSlot = kScaleGroups * kTaTile * 4;
constexpr int kTaSlot = kNopeSlot + kRopeSlot + kScaleSlot;  // nope bytes, rope, scales [group][token] of a tile

// LDS of a workgroup with R row groups: the ring's slots [slot][stream]; the query's rope fragments; per wave and
// row visibility bits, later the softmax's state; per wave what its registers have no room for while it
// works on the next tile's logits. The merge of two streams takes the ring's place at the end.
template <int R>
struct TaLds {
    static constexpr int kStreams = kTaWaves / R;
    static constexpr int kQuery = kStreams * kTaSlots * kTaSlot;
    static constexpr int kState = kQuery + R * 4096;
    static constexpr int kKept = kState + kTaWaves * kTaRows * 8;  // per wave a tile's probabilities
    static constexpr int kBytes = kKept + kTaWaves * 4096;
    static constexpr int kMerge = kTaWaves * 4 * 4096;  // 4 blocks of 4 KB per wave
    static_assert(kBytes <= 160 * 1024, "LDS of a CU");
    static_assert(kStreams == 1 || kMerge <= kQuery, "merge buffer in the ring");
};

__host__ __device__ inline int ta_tiles(int rows, int r) { return (rows + kTaRows * r - 1) / (kTaRows * r); }

// Row groups R. Four halve the cache rows that a workgroup reads per product, two waste less where the rows do not
// fill a last tile of 128: a row's step costs 1.08 times as much with two (128 heads x 12 tokens on 2000-8192
// cache rows: 227 us, 210 with four), so they pay where they save one of at most 12 half tiles (32 heads x 9
// tokens on 131000 cache rows: 231 to 255 us, as the cache lies in memory, 254 with four).
inline int ta_groups(int heads, int nodes) {
    const int halves = ta_tiles(heads * nodes, 2), full = 2 * ta_tiles(heads * nodes, 4);
    return halves * 13 < full * 12 ? 2 : 4;
}

// Steps of a launch at most (the kernel counts them in 32 bits), and its shares: one workgroup per CU, no more
// than these steps could fill.
inline int64_t ta_most_steps(int batch, int heads, int nodes, int max_blocks) {
    const int r = ta_groups(heads, nodes), streams = kTaWaves / r;
    const int64_t steps = (static_cast<int64_t>(max_blocks) * kBlockTokens + kTaTile * streams - 1) / (kTaTile * streams) + kHeadSteps;
    return steps * batch * ta_tiles(heads * nodes, r);
}
inline int ta_shares(int batch, int heads, int nodes, int max_blocks) {
    const int64_t most = (ta_most_steps(batch, heads, nodes, max_blocks) + kMinSteps - 1) / kMinSteps;
    return static_cast<int>(most < kTaGroups ? most : kTaGroups);
}

// x, recomputed from here on: keeps the compiler from holding dozens of addresses over the tile loop.
KVIP_DEVICE int fresh(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

KVIP_DEVICE uint32_t pack_bf16(float a, float b) {  // hardware round to nearest even
    const bf16x2 v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
    return __builtin_bit_cast(uint32_t, v);
}

// Eight fp8 e4m3 features as bf16 (exact).
KVIP_DEVICE bf16x8 fp8x8_to_bf16(int lo, int hi) {
    const v4i r = {
        __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false)),
        __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true)),
        __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false)),
        __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true))};
    return __builtin_bit_cast(bf16x8, r);
}

KVIP_DEVICE float half_max(float x) {  // over lanes l and l ^ 32
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
KVIP_DEVICE float half_sum(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// Places of a token's 16-byte pieces in its 512-byte LDS row: piece j sits at place j ^ swz(token).
// Linear over XOR; a key read (16 consecutive lanes: one piece of 16 consecutive tokens) and a
// value read (32 lanes: two neighbouring pieces of 8 tokens that differ in bits 0, 1 and 3) each touch
// every bank once.
KVIP_DEVICE constexpr int ta_swz(int t) { return ((t >> 2) & 1) | ((t & 1) << 1) | ((t & 2) << 1) | (t & 8); }

// Where the workspace holds what: per share two parts (its first item's, where others began it, and its
// last one's, where others go on) of 32 R rows x 512 sums as a wave's lanes hold them ([row group][block][quarter]
// [lane] 16 bytes: stored and read whole lines at a time), their (maximum, sum) pairs, then per item the first
// share and the number of shares.
template <int R>
struct TaWork {
    f32x4* sums;
    float2* state;
    int2* items;
    KVIP_DEVICE TaWork(void* base, int shares) {
        sums = static_cast<f32x4*>(base);
        state = reinterpret_cast<float2*>(sums + static_cast<size_t>(shares) * 2 * R * (kBlocks * 4 * 64));
        items = reinterpret_cast<int2*>(state + static_cast<size_t>(shares) * 2 * R * kTaRows);
    }
    // Group `rg` of a part's rows: its sums (of lane 0) and states.
    KVIP_DEVICE f32x4* group(int part, int rg) const { return sums + (static_cast<size_t>(part) * R + rg) * (kBlocks * 4 * 64); }
    KVIP_DEVICE float2* rows(int part, int rg) const { return state + (static_cast<size_t>(part) * R + rg) * kTaRows; }
};

// log sum_j exp(s_j) of a row: maximum in log2 units, sum (0 where the row sees nothing).
KVIP_DEVICE float ta_lse(float m, float l) {
    return l > 0.f || l != l ? (m + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
}

// Four features of the output.
KVIP_DEVICE void ta_store(const KvipTreeAttnArgs& p, int64_t at, f32x4 v) {
    if (p.output_dtype == KVIP_DTYPE_FP32) {
        *reinterpret_cast<f32x4*>(static_cast<float*>(p.output) + at) = v;
    } else {
        *reinterpret_cast<bf16x4*>(static_cast<__bf16*>(p.output) + at) = __builtin_convertvector(v, bf16x4);
    }
}

// Barrier for LDS data: unlike __syncthreads it leaves the direct-to-LDS loads in flight.
KVIP_DEVICE void lds_sync() {
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
}

// A request as the kernel takes it.
struct TaRequest {
    int begin;   // first row of the step
    int nodes;   // its step tokens (at most max_nodes)
    int past;    // position of step token 0 (below 0 where the length is too short)
    int length;  // cache rows (a refused request's: none, so that its rows get their zeros)
};

KVIP_DEVICE TaRequest ta_request(const KvipTreeAttnArgs& p, int b, uint32_t* err) {
    TaRequest q;
    const int first = p.cu_seqlens[b], behind = p.cu_seqlens[b + 1];
    q.begin = min(max(first, 0), p.max_tokens);
    const int all = min(max(behind, q.begin), p.max_tokens) - q.begin;
    const int given = p.seq_lens[b];
    const bool refused = p.steps != nullptr && p.steps[b] <= 0;
    q.nodes = min(all, p.max_nodes);
    q.length = refused ? 0 : min(max(given, 0), p.max_blocks * kBlockTokens);
    q.past = q.length - all;
    if (first != q.begin || behind != q.begin + all) *err |= KVIP_STATUS_BAD_LENGTH;
    if (all != q.nodes || (!refused && (given != q.length || (all > 0 && q.past < 0)))) *err |= KVIP_STATUS_BAD_LENGTH;
    return q;
}

// Steps of an item: at least one, so that rows without any token get their zeros.
template <int R>
KVIP_DEVICE int ta_steps(int length) {
    constexpr int kTokens = kTaTile * (kTaWaves / R);
    return max((length + kTokens - 1) / kTokens, 1);
}

// Direct-to-LDS loads from a wave-uniform address and a lane's offset below 2^32 (see lds_async.h).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
KVIP_DEVICE void dma16_at(const uint8_t* base, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds), "v"(offset), "s"(base) : "memory", "m0");
}
KVIP_DEVICE void dma4_at(const uint8_t* base, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" : : "s"(lds), "v"(offset), "s"(base) : "memory", "m0");
}
#pragma clang diagnostic pop

// Keeps an accumulator in accumulation registers from here to the next hold: left to itself the compiler
// moves parts of the 256 between the two halves of the register file in every tile.
KVIP_DEVICE void hold(v16f& acc) { asm volatile("" : "+a"(acc)); }

template <int R>
__global__ __launch_bounds__(kTaThreads, 1) void tree_attention_kernel(const KvipTreeAttnArgs p) {
    typedef TaLds<R> L;
    constexpr int kStreams = L::kStreams;
    __shared__ __align__(1024) uint8_t s_mem[L::kBytes];
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rg = w % R, st = w / R;  // row group, stream
    const int shares = gridDim.x;
    // Neighbouring shares, which read the same cache rows where an item or a request spans them, on one
    // XCD (workgroups are dealt round the 8).
    const int per_xcd = shares / 8;
    const int g = static_cast<int>(blockIdx.x) < per_xcd * 8 ? static_cast<int>(blockIdx.x % 8) * per_xcd + blockIdx.x / 8
                                                             : blockIdx.x;

    // The line of work, 4 requests per thread: an item's length in it, and this share's part [pos, end), from
    // request b, which starts at b_pos. It is laid out in one of two ways, whichever gives shares the less to do:
    //   - Few items: each is cut on its own into shares of `quota` steps, its length a multiple of that.
    //   - Else they stand one after the other, each with what its start costs (`head`) before its steps, as shares
    //     that start many would end last; a cut within `near` steps of an item's start or end moves there.
    // (17 requests of 2 tokens, 8 heads, 1-141 rows took 33 us with all items in one line, cut anywhere.)
    int b;
    uint32_t pos, end, b_pos, quota, head, near;
    bool apart;
    TaRequest req;
    {
        constexpr int kPer = KVIP_DRAFT_MAX_BATCH / kTaThreads;
        uint32_t* s_sum = reinterpret_cast<uint32_t*>(s_mem);
        uint32_t* s_items = s_sum + kTaWaves;
        int* s_found = reinterpret_cast<int*>(s_items + kTaWaves);  // request, where it starts, what it is
        const int per = (p.batch + kTaThreads - 1) / kTaThreads;  // requests of a thread, at most kPer
        TaRequest of[kPer];
        uint32_t tiles[kPer], steps[kPer], sum = 0, items = 0, err = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int at = tid * per + i;
            tiles[i] = steps[i] = 0;
            if (i < per && at < p.batch) {
                of[i] = ta_request(p, at, &err);
                tiles[i] = ta_tiles(of[i].nodes * p.heads, R);
                steps[i] = ta_steps<R>(of[i].length);
            }
            items += tiles[i];
            sum += tiles[i] * steps[i];
        }
        if (blockIdx.x == 0) report(p.status, err);
        const uint32_t run = wave_inclusive_scan(sum), run_items = wave_inclusive_scan(items);
        if (lane == 63) {
            s_sum[w] = run;
            s_items[w] = run_items;
        }
        __syncthreads();
        uint32_t before = run - sum, before_items = run_items - items, total = 0, all_items = 0;
#pragma unroll
        for (int v = 0; v < kTaWaves; ++v) {
            before += v < w ? s_sum[v] : 0u;
            before_items += v < w ? s_items[v] : 0u;
            total += s_sum[v];
            all_items += s_items[v];
        }
        const uint32_t in_line = (total + kHeadSteps * all_items + shares - 1) / shares;
        const uint32_t left = all_items < static_cast<uint32_t>(shares) ? shares - all_items : 0;
        const uint32_t of_item = left == 0 ? 0 : max((total + left - 1) / left, static_cast<uint32_t>(kMinSteps));
        apart = left != 0 && of_item <= max(in_line, static_cast<uint32_t>(kMinSteps));
        quota = apart ? of_item : in_line;
        head = apart ? 0 : kHeadSteps;
        near = apart || total >= 4 * kHeadSteps * all_items ? 0 : quota / 16;  // short items, which a cut costs most
        if (apart) {
            uint32_t cuts = 0;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                if (i >= per) break;
                steps[i] = (steps[i] + quota - 1) / quota;
                cuts += tiles[i] * steps[i];
                steps[i] *= quota;
            }
            const uint32_t run_cuts = wave_inclusive_scan(cuts);
            __syncthreads();  // the sums before are read
            if (lane == 63) s_sum[w] = run_cuts;
            __syncthreads();
            before = run_cuts - cuts;
            total = 0;
#pragma unroll
            for (int v = 0; v < kTaWaves; ++v) {
                before += v < w ? s_sum[v] : 0u;
                total += s_sum[v];
            }
            before *= quota;
            total *= quota;
        } else {
            before += head * before_items;
            total += head * all_items;
        }
        pos = min(g * quota, total);
        end = min(pos + quota, total);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const uint32_t cost = tiles[i] * (steps[i] + head);
            if (before <= pos && pos < before + cost) {
                s_found[0] = tid * per + i;
                s_found[1] = before;
                *reinterpret_cast<TaRequest*>(s_found + 2) = of[i];
            }
            before += cost;
        }
        __syncthreads();
        if (pos >= end) return;  // the whole workgroup: more shares than steps
        b = __builtin_amdgcn_readfirstlane(s_found[0]);
        b_pos = __builtin_amdgcn_readfirstlane(s_found[1]);
        const TaRequest* found = reinterpret_cast<const TaRequest*>(s_found + 2);
        req.begin = __builtin_amdgcn_readfirstlane(found->begin);
        req.nodes = __builtin_amdgcn_readfirstlane(found->nodes);
        req.past = __builtin_amdgcn_readfirstlane(found->past);
        req.length = __builtin_amdgcn_readfirstlane(found->length);
    }
    const TaWork<R> work(p.workspace, shares);
    const uint32_t ring_lds = lds_addr(s_mem) + st * kTaSlot;
    // Logits are kept as they come and scaled on their way into the exponential. A negative scale turns the
    // query's signs; one of 0 becomes 2^-126, which no logit below 10^32 shows.
    const float scale2 = __int_as_float(__builtin_amdgcn_readfirstlane(
        __float_as_int(fmaxf(fabsf(p.scale * kLog2e), 0x1p-126f))));
    const int flip = p.scale < 0.f ? static_cast<int>(0x80008000u) : 0;
    const int row_stride = p.row_stride;

    while (pos < end) {
        // The item at `pos`: request b, row tile rt, steps t0 .. t1 of its `steps`, which stand behind its head.
        uint32_t err = 0;
        auto length_of = [&](uint32_t steps) { return apart ? (steps + quota - 1) / quota * quota : steps + head; };
        auto cost_of = [&](const TaRequest& q) {
            return static_cast<uint32_t>(ta_tiles(q.nodes * p.heads, R)) * length_of(ta_steps<R>(q.length));
        };
        uint32_t cost = cost_of(req);
        // Ends at the request that holds pos, as pos < end <= the line's length.
        while (pos >= b_pos + cost && b + 1 < p.batch) {
            b_pos += cost;
            req = ta_request(p, ++b, &err);
            cost = cost_of(req);
        }
        err = 0;
        const int steps = ta_steps<R>(req.length), length = length_of(steps);
        const uint32_t within = min(pos - b_pos, max(cost, 1u) - 1);
        const int rt = __builtin_amdgcn_readfirstlane(within / length);
        const int from_at = __builtin_amdgcn_readfirstlane(within - rt * length);
        const int to_at = __builtin_amdgcn_readfirstlane(min(length, static_cast<int>(from_at + (end - pos))));
        const uint32_t item_pos = pos - from_at;
        pos += to_at - from_at;
        // Step of a cut of the line.
        auto cut = [&](int at) {
            const int t = at - static_cast<int>(head);
            return at == length ? steps : t <= static_cast<int>(near) ? 0 : t + static_cast<int>(near) >= steps ? steps : t;
        };
        const int t0 = from_at == 0 ? 0 : cut(from_at), t1 = cut(to_at);
        if (t0 >= t1) continue;  // others have it
        const bool whole = t0 == 0 && t1 == steps;
        const int rows = req.nodes * p.heads;
        const int first_row = rt * kTaRows * R + rg * kTaRows;
        const bool busy = first_row < rows;  // uniform: the wave's group has rows
        const int32_t* table = p.block_table + static_cast<int64_t>(b) * p.max_blocks;

        // Page of the wave's tile of step t (-1: none of its tokens is there), from the table entries of 64 pages
        // that the lanes hold.
        int held_first = t0 * kStreams / (kBlockTokens / kTaTile);
        int held = table[min(held_first + lane, p.max_blocks - 1)];
        auto page_of = [&](int t) {
            const int tile = t * kStreams + st, at = tile / (kBlockTokens / kTaTile);
            if (tile * kTaTile >= req.length) return -1;
            if (at >= held_first + 64) {
                held_first = at;
                held = table[min(at + lane, p.max_blocks - 1)];
                asm volatile("" : "+v"(held));  // waited for here, not at every use
            }
            const int page = __builtin_amdgcn_readlane(held, at - held_first);
            if (static_cast<unsigned>(page) < static_cast<unsigned>(p.num_blocks)) return page;
            err |= KVIP_STATUS_BAD_BLOCK;
            return -1;
        };
        // The tile to load: the first row of this wave's share (1 / R) of its tokens, and its LDS slot. A tile is
        // part of one page, so its 32 rows are in the cache, whatever the length; where there is no page the
        // cache's first ones stand in. `logits` zeroes in LDS what is not there.
        constexpr int kShare = kTaTile / R, kPageSteps = kBlockTokens / (kTaTile * kStreams);
        const uint8_t *tile_from, *from;
        uint32_t to, to_rope;
        auto into = [&](uint32_t slot) {
            from = tile_from;
            to = slot + rg * (kShare * kValueDim);
            to_rope = slot + kNopeSlot + rg * (kShare * 128);
            asm volatile("" : "+s"(to), "+s"(to_rope));
        };
        auto aim = [&](int t, int page) {
            const int first = (t * kStreams + st) % (kBlockTokens / kTaTile) * kTaTile;
            tile_from = p.kv_cache + max(page, 0) * p.kv_block_stride + static_cast<int64_t>(first + rg * kShare) * row_stride;
        };
        // The share's loads, in kFetches pieces that are called in order. LDS row i of the nope bytes holds piece
        // s ^ ta_swz(i) at place s, of the rope features (128 bytes) piece s ^ (i / 2 % 8); scales stand as
        // [group][token].
        constexpr int kNopeLoads = kShare / 2, kRopeLoads = kShare / 8, kFetches = kNopeLoads + kRopeLoads + 1;
        constexpr int kEvery = 16 / kFetches;  // products of the logits from one piece to the next
        auto fetch = [&](int x, int ln) {
            if (x < kNopeLoads) {  // the share's tokens 2 x and 2 x + 1 (ta_swz is linear over XOR)
                const int up = ln >> 5;
                dma16_at(from, up * row_stride + ((ln & 31) ^ ta_swz(up) ^ ta_swz(rg * kShare) ^ ta_swz(2 * x)) * 16,
                         to + x * 1024);
                from += x + 1 < kNopeLoads ? 2 * row_stride : -(2 * kNopeLoads - 2) * row_stride;
            } else if (x < kNopeLoads + kRopeLoads) {  // tokens 8 y .. 8 y + 7
                const int y = x - kNopeLoads, v = rg * kRopeLoads + y;
                dma16_at(from, (ln >> 3) * row_stride + kValueDim + ((ln & 7) ^ (ln >> 4) ^ ((v & 1) * 4)) * 16,
                         to_rope + y * 1024);
                from += y + 1 < kRopeLoads ? 8 * row_stride : -(8 * kRopeLoads - 8 + rg * kShare) * row_stride;
            } else {  // scale groups 2 v and 2 v + 1 of all tokens (with 4 row groups, two of them load the same)
                const int v = rg & 1;
                dma4_at(from + 8 * v, (ln & 31) * row_stride + 640 + 4 * (ln >> 5), to_rope + (kRopeSlot - rg * (kShare * 128) + v * 256));
            }
        };
        // Every load and LDS access of this wave is done, and of all waves.
        auto settle = [&] {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" : : : "memory");
        };

        lds_sync();  // the LDS of the item before (at first: the line of work) is free; its stores may be under way
        int page = page_of(t0), page_next = page;
        aim(t0, page);
        into(ring_lds);
#pragma unroll
        for (int x = 0; x < kFetches; ++x) fetch(x, lane);
        // Step t: its tile has landed, and the slot of step t - 2's is free for that of step t + 1 (the last step loads
        // its own again).
        auto arrive = [&](int t, uint32_t slot_free) {
            settle();
            page = page_next;
            if (t + 1 < t1) {
                if ((t + 1) % kPageSteps == 0) {
                    page_next = page_of(t + 1);
                    aim(t + 1, page_next);
                } else {
                    tile_from += kTaTile * kStreams * row_stride;
                }
            }
            into(slot_free);
        };
        // Steps with step tokens or the end of the context in them (the same for the workgroup's waves).
        const int t_last = max(req.past, 0) / (kStreams * kTaTile);
        constexpr int kSlotStep = kStreams * kTaSlot;
        if (!busy) {  // a row group without rows loads its share of the tiles
            for (int t = t0; t < t1; ++t) {
                arrive(t, ring_lds + (t + 1 - t0) % kTaSlots * kSlotStep);
                if (t >= t_last) lds_sync();
#pragma unroll
                for (int x = 0; x < kFetches; ++x) fetch(x, lane);
            }
            asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // the loads past the last tile
            if constexpr (kStreams > 1) {  // the barriers of the merge
                for (int i = 0; i < 5; ++i) lds_sync();
            }
        } else {
            const uint32_t rope_q_lds = lds_addr(s_mem + L::kQuery) + rg * 4096;                 // + lane * 16
            uint64_t* s_seen = reinterpret_cast<uint64_t*>(s_mem + L::kState) + w * kTaRows;  // + row of the wave
            // Queries of the wave's rows (rows past the last read it again; their outputs are not written). Fragment
            // 2 i + x: features 16 (2 i + kg) + 8 x .. + 7, the half x of the key piece that the lane reads; rope
            // fragment i: features 16 i + 8 kg .. + 7.
            const int at = min(first_row + (lane & 31), rows - 1), node = at / p.heads;
            const uint16_t* q = p.query + (static_cast<int64_t>(req.begin) * p.heads + at) * kKeyDim + (lane >> 5) * 8;
            v4i qf[32], q_rope[4];
#pragma unroll
            for (int i = 0; i < 32; ++i) qf[i] = *reinterpret_cast<const v4i*>(q + (i >> 1) * 32 + (lane >> 5) * 8 + (i & 1) * 8);
#pragma unroll
            for (int i = 0; i < 4; ++i) q_rope[i] = *reinterpret_cast<const v4i*>(q + kValueDim + i * 16);
            const uint64_t seen_by =
                p.visible != nullptr ? static_cast<uint64_t>(p.visible[req.begin + node]) : ~0ull >> (63 - node);
            v16f o[kBlocks];
#pragma unroll
            for (int f = 0; f < kBlocks; ++f) {
#pragma unroll
                for (int i = 0; i < 16; ++i) o[f][i] = 0.f;
                hold(o[f]);
            }
            // Waited for here: the tile loop would wait for them each time round, and so for its own loads.
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                qf[i] ^= flip;
                asm volatile("" : "+v"(qf[i]));
            }
            float m_run = -INFINITY;  // reference maximum of the row
            float l_sum = 0.f;        // this lane's share of its probability sum
            // Probabilities of the tile whose values come next, relative to m_run: in LDS while the logits need the registers.
            const uint32_t kept_lds = lds_addr(s_mem + L::kKept) + w * 4096;
            v16f s;                   // logits

            auto landed = [] { __builtin_amdgcn_s_waitcnt(0xC07F); };  // lgkmcnt(0): one wait for the reads before
            constexpr int kAhead = 3;  // LDS reads stand two or three products before their use, in pairs, conversions one
            // Logits of step t's tile, in slot `slot`; the loads of the tile that is aimed at stand between the products.
            auto logits = [&](int t, uint32_t slot) {
                const int ln = fresh(lane), tn = ln & 31, tk = ln >> 5;
                const int first = (t * kStreams + st) * kTaTile;  // position of the tile's first token
                uint32_t sees = page < 0 ? 0u : 0xFFFFu;          // bit i: the row sees the token of register i
                bool masked = page < 0;
                // A step of the last, or a tile that is not there. What a row does not see must not reach it, and zero times a NaN would:
                // tokens that are not there, and those with a NaN feature or a scale that is not finite, are
                // zeroed in LDS, and rows that do see one of the latter become NaN as a whole (their logit is none).
                if (masked || t >= t_last) {
                    masked = true;
                    uint32_t nan = 0;
                    const uint32_t at = slot + tn * kValueDim;
                    const uint32_t sc = slot + kNopeSlot + kRopeSlot + tk * 2 * kTaTile * 4 + tn * 4;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const v4i x = *(LdsV4i)(at + (((16 * tk + i) ^ ta_swz(tn)) << 4));
#pragma unroll
                        for (int e = 0; e < 4; ++e) nan |= (x[e] & 0x7F7F7F7Fu) + 0x01010101u;
                    }
                    nan &= 0x80808080u;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t x = __float_as_uint(*(LdsF32)(sc + i * kTaTile * 4));
                        nan |= (x & 0x7F800000u) == 0x7F800000u ? 1u : 0u;
                    }
                    const uint64_t found = __ballot(nan != 0);
                    const uint32_t bad = static_cast<uint32_t>(found | found >> 32);
                    if (t >= t_last) lds_sync();  // the waves of the stream have all looked (or none needs to)
                    if ((bad >> tn & 1) || page < 0 || first + tn >= req.length) {
#pragma unroll 4
                        for (int i = 0; i < 16; ++i) {
                            *(__attribute__((address_space(3))) v4i*)(at + (16 * tk + i) * 16) = v4i{0, 0, 0, 0};
                        }
#pragma unroll
                        for (int i = 0; i < 2; ++i) *(__attribute__((address_space(3))) float*)(sc + i * kTaTile * 4) = 0.f;
                    }
                    // Bit j: the row sees the tile's token j. The step's token 0 is the tile's token -d.
                    const uint64_t seen = s_seen[tn];
                    const int d = first - req.past, left = req.length - first;
                    uint32_t row_sees = d >= 64 ? 0u : d >= 0 ? static_cast<uint32_t>(seen >> d) : d > -32 ?
                        static_cast<uint32_t>(seen) << -d | ((1u << -d) - 1) : ~0u;
                    if (left < 32) row_sees &= left <= 0 ? 0u : (1u << left) - 1;
                    if (page < 0) row_sees = 0;
                    if (row_sees & bad) l_sum = NAN;
                    row_sees >>= 4 * tk;
                    sees = (row_sees & 0xF) | (row_sees >> 4 & 0xF0) | (row_sees >> 8 & 0xF00) | (row_sees >> 12 & 0xF000);
                }
                const uint32_t ro = slot + kNopeSlot + tn * 128 + ((tk ^ ((tn >> 1) & 7)) << 4);
                uint32_t ko = slot + tn * kValueDim + ((tk ^ ta_swz(tn)) << 4);
                const uint32_t sl = slot + kNopeSlot + kRopeSlot + 16 * tk;  // scales of tokens 8 a + 4 kg .. + 3
                // Bit 8 of a key's address is its own: pieces 16 and up by an offset.
                auto key = [&](int i) { return *(LdsV4i)((ko ^ ((i & 7) * 32)) + (i >> 3) * 256); };
                v16f dot[2];
                // A quarter of a group's dot products (tokens 8 a + 4 kg .. + 3) joins the logits a group later, its
                // scales are read a little before that.
                f32x4 s4[16];
                auto scales = [&](int q) { s4[q] = *(LdsF32x4)(sl + ((q >> 2) * kTaTile + 8 * (q & 3)) * 4); };
                auto join = [&](int q) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int e = 4 * (q & 3) + c;
                        s[e] = fmaf(dot[q >> 2 & 1][e], s4[q][c], s[e]);
                    }
                };
                {
                    v4i kb[kAhead + 1];
                    {
                        const uint32_t yo = fresh(rope_q_lds + ln * 16);
                        v4i kr[4], yr[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            kr[i] = *(LdsV4i)(ro ^ (i * 32));
                            yr[i] = *(LdsV4i)(yo + i * 1024);
                        }
#pragma unroll
                        for (int i = 0; i < kAhead; ++i) kb[i] = key(i);
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, kr[i]), __builtin_bit_cast(bf16x8, yr[i]), s, 0, 0, 0);
                        }
                    }
                    bf16x8 ka[2] = {fp8x8_to_bf16(kb[0][0], kb[0][1]), fp8x8_to_bf16(kb[0][2], kb[0][3])};
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int gr = i >> 2;
                        v16f& d = dot[gr & 1];
                        if ((i & 3) == 0) {
#pragma unroll
                            for (int e = 0; e < 16; ++e) d[e] = 0.f;
                        }
                        d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[0], __builtin_bit_cast(bf16x8, qf[2 * i]), d, 0, 0, 0);
                        if ((i & 1) == 0) {
                            landed();
                            if (i >= 4) {
                                scales(i - 4);
                                scales(i - 3);
                            }
#pragma unroll
                            for (int k = i + kAhead; k < i + kAhead + 2 && k < 16; ++k) {
                                if (k == 8) ko = fresh(ko);  // rather than hold eight addresses
                                kb[k % (kAhead + 1)] = key(k);
                            }
                        }
                        const v4i x = kb[(i + 1) % (kAhead + 1)];
                        if (i < 15) ka[0] = fp8x8_to_bf16(x[0], x[1]);
                        if (i % kEvery == 0 && i / kEvery < kFetches) fetch(i / kEvery, ln);
                        __builtin_amdgcn_sched_barrier(0);
                        d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[1], __builtin_bit_cast(bf16x8, qf[2 * i + 1]), d, 0, 0, 0);
                        if (i < 15) ka[1] = fp8x8_to_bf16(x[2], x[3]);
                        if (i >= 4 && (i & 1) == 1) {
                            join(i - 5);
                            join(i - 4);
                        }
                        if (i == 15) {
#pragma unroll
                            for (int q = 12; q < 16; ++q) scales(q);
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
#pragma unroll
                for (int q = 12; q < 16; ++q) join(q);
                if (masked) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        if (!(sees >> i & 1)) s[i] = -INFINITY;
                    }
                }
            };
            // Softmax of the logits, p = 2^(scale2 (logit - m)), in 18 pieces. Its factor for what came before (alpha)
            // counts once the values of the tile before are in.
            float mx, bias, alpha, fresh_sum;
            bool raise;
            auto softmax = [&](int piece) {
                if (piece == 0) {
                    mx = s[0];
#pragma unroll
                    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
                    mx = half_max(mx);
                    fresh_sum = 0.f;
                } else if (piece == 1) {
                    raise = (mx - m_run) * scale2 > kTaMargin;  // also the first finite maximum
                    const float m_new = raise ? mx : m_run;
                    alpha = raise && m_run != -INFINITY ? __builtin_amdgcn_exp2f((m_run - m_new) * scale2) : raise ? 0.f : 1.f;
                    m_run = m_new;
                    bias = m_new == -INFINITY ? 0.f : -m_new * scale2;
                } else {
                    s[piece - 2] = __builtin_amdgcn_exp2f(fmaf(s[piece - 2], scale2, bias));
                    fresh_sum += s[piece - 2];
                    if ((piece & 1) == 1) asm volatile("" : "+v"(fresh_sum));  // here, not behind the products
                }
            };
            auto take = [&] {  // the softmax's results become those of the tile whose values come next
                l_sum = l_sum * alpha + fresh_sum;
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    *(LdsF32x4Out)(kept_lds + fresh(lane) * 16 + a * 1024) = f32x4{s[4 * a], s[4 * a + 1], s[4 * a + 2], s[4 * a + 3]};
                }
            };
            // Values of the tile in slot `slot` [features, rows], the softmax of the next one beside them.
            auto values = [&](uint32_t slot, auto with_softmax) {
                constexpr bool kSoftmax = decltype(with_softmax)::value;
                const int ln = fresh(lane), tk = ln >> 5;
                const int y = (ln & 15) >> 1, vt = 8 * (y >> 2) + 4 * tk + (y & 3);
                const uint32_t vo = slot + vt * kValueDim + ((((ln >> 4) & 1) ^ ta_swz(vt)) << 4) + 8 * (ln & 1);
                const uint32_t sl = slot + kNopeSlot + kRopeSlot + 16 * tk;
                auto value = [&](int f, int h) {
                    return __builtin_amdgcn_ds_read_tr8_b64_v2i32((LdsI32x2)((vo ^ ((f & 7) * 32)) + (f >> 3) * 256 + h * 16 * kValueDim));
                };
                // A quarter of a group's operand: the probabilities of tokens 8 a + 4 kg .. + 3 times their scales, which
                // are read two products earlier.
                v4i pb[2][2];
                f32x4 s4[4], pr[4];
                auto scales = [&](int q) { s4[q & 3] = *(LdsF32x4)(sl + ((q >> 2) * kTaTile + 8 * (q & 3)) * 4); };
                auto weigh = [&](int q) {
                    const int a = q & 3;
                    v4i& d = pb[q >> 2 & 1][a >> 1];
                    d[2 * (a & 1)] = static_cast<int>(pack_bf16(pr[a][0] * s4[a][0], pr[a][1] * s4[a][1]));
                    d[2 * (a & 1) + 1] = static_cast<int>(pack_bf16(pr[a][2] * s4[a][2], pr[a][3] * s4[a][3]));
                };
                i32x2 vb[kAhead + 1][2];
#pragma unroll
                for (int a = 0; a < 4; ++a) pr[a] = *(LdsF32x4)(kept_lds + ln * 16 + a * 1024);
#pragma unroll
                for (int q = 0; q < 4; ++q) scales(q);
#pragma unroll
                for (int f = 0; f < kAhead; ++f) {
                    vb[f][0] = value(f, 0);
                    vb[f][1] = value(f, 1);
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) weigh(q);
                bf16x8 va[2] = {fp8x8_to_bf16(vb[0][0][0], vb[0][0][1]), fp8x8_to_bf16(vb[0][1][0], vb[0][1][1])};
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int f = 0; f < kBlocks; ++f) {
                    const int gr = f >> 2, next = (f + 1) % (kAhead + 1);
                    hold(o[f]);
                    o[f] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va[0], __builtin_bit_cast(bf16x8, pb[gr & 1][0]), o[f], 0, 0, 0);
                    if ((f & 1) == 0) {
                        landed();
#pragma unroll
                        for (int q = f + 4; q < f + 6 && q < 16; ++q) scales(q);
#pragma unroll
                        for (int k = f + kAhead; k < f + kAhead + 2 && k < kBlocks; ++k) {
                            vb[k % (kAhead + 1)][0] = value(k, 0);
                            vb[k % (kAhead + 1)][1] = value(k, 1);
                        }
                    }
                    if (f + 1 < kBlocks) va[0] = fp8x8_to_bf16(vb[next][0][0], vb[next][0][1]);
                    if (kSoftmax) softmax(f);
                    __builtin_amdgcn_sched_barrier(0);
                    o[f] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va[1], __builtin_bit_cast(bf16x8, pb[gr & 1][1]), o[f], 0, 0, 0);
                    hold(o[f]);
                    if (f + 1 < kBlocks) va[1] = fp8x8_to_bf16(vb[next][1][0], vb[next][1][1]);
                    if ((f & 1) == 1) {
#pragma unroll
                        for (int q = f + 3; q < f + 5 && q < 16; ++q) weigh(q);
                    }
                    if (kSoftmax && f == kBlocks - 1) {
                        softmax(16);
                        softmax(17);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            };

            uint32_t slot = ring_lds, slot_next = ring_lds + kSlotStep, slot_free = ring_lds + 2 * kSlotStep;
            arrive(t0, slot_next);
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // the streams of a row group write the same
                *(__attribute__((address_space(3))) v4i*)(rope_q_lds + fresh(lane) * 16 + i * 1024) = q_rope[i] ^ flip;
            }
            s_seen[lane & 31] = seen_by;
            logits(t0, slot);
#pragma unroll
            for (int i = 0; i < 18; ++i) softmax(i);
            take();
#pragma unroll 1
            for (int t = t0; t + 1 < t1; ++t) {
                arrive(t + 1, slot_free);
                logits(t + 1, slot_next);
                values(slot, std::true_type{});
                if (__ballot(raise) != 0ull) {
#pragma unroll
                    for (int f = 0; f < kBlocks; ++f) {
                        hold(o[f]);  // read here, not in every tile
                        o[f] *= alpha;
                        hold(o[f]);
                    }
                }
                take();
                const uint32_t used = slot;
                slot = slot_next;
                slot_next = slot_free;
                slot_free = used;
            }
            values(slot, std::false_type{});
            asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // the loads past the last tile
            // A seen scale that is not finite: where it made a logit -infinity, the probability 0 times the scale left
            // NaN in all of the scale group's features, but in no other.
#pragma unroll
            for (int gr = 0; gr < kScaleGroups; ++gr) {
                hold(o[4 * gr]);
                if (o[4 * gr][0] != o[4 * gr][0]) l_sum = NAN;
            }

            const int le = fresh(lane), hn = le & 31, hk = le >> 5;  // not held over the tiles
            const int row = first_row + hn;
            const int64_t out_row = static_cast<int64_t>(req.begin) * p.heads + row;
            const int part = g * 2 + (t0 == 0 ? 1 : 0);
            // A whole item's rows are final; else the sums and their state go to the share's part 0 (others began
            // the item) or 1.
            auto put = [&](int f, const v16f& x, float factor) {
                if (!whole) {
                    f32x4* out = work.group(part, rg) + le;
#pragma unroll
                    for (int a = 0; a < 4; ++a) out[(f * 4 + a) * 64] = f32x4{x[4 * a], x[4 * a + 1], x[4 * a + 2], x[4 * a + 3]};
                    return;
                }
                if (p.output_dtype == KVIP_DTYPE_BF16) {
                    // The halves of the wave hold every other four features of a row: swapped, each has eight.
#pragma unroll
                    for (int a = 0; a < 4; a += 2) {
                        v4i v;
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const auto pair = __builtin_amdgcn_permlane32_swap(
                                pack_bf16(x[4 * a + 2 * e] * factor, x[4 * a + 2 * e + 1] * factor),
                                pack_bf16(x[4 * a + 2 * e + 4] * factor, x[4 * a + 2 * e + 5] * factor), false, false);
                            v[e] = pair[0];
                            v[e + 2] = pair[1];
                        }
                        if (row < rows) *reinterpret_cast<v4i*>(static_cast<__bf16*>(p.output) + out_row * kValueDim + 32 * f + 8 * a + 8 * hk) = v;
                    }
                    return;
                }
                if (row >= rows) return;
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    const f32x4 v = f32x4{x[4 * a], x[4 * a + 1], x[4 * a + 2], x[4 * a + 3]} * factor;
                    ta_store(p, out_row * kValueDim + 32 * f + 8 * a + 4 * hk, v);
                }
            };
            auto put_state = [&](float m, float l) {
                if (st != 0 || hk != 0) return;
                if (!whole) work.rows(part, rg)[hn] = make_float2(m, l);
                else if (p.lse != nullptr && row < rows) p.lse[out_row] = ta_lse(m, l);
            };
            const float l_all = half_sum(l_sum);
            const float m_all = m_run * scale2;  // log2 units from here on
            if constexpr (kStreams == 1) {
                const float factor = whole ? (l_all > 0.f || l_all != l_all ? 1.f / l_all : 0.f) : 1.f;
#pragma unroll
                for (int f = 0; f < kBlocks; ++f) {
                    hold(o[f]);
                    put(f, o[f], factor);
                }
                put_state(m_all, l_all);
            } else {
                // Merge of the two streams: with the maximum M over them, sums = sum_w 2^(m_w - M) o_w and l likewise. A
                // wave sums half of the blocks, whose other half it puts into LDS, 8 blocks at a time.
                float2* s_state = reinterpret_cast<float2*>(s_mem + L::kState);
                lds_sync();  // every wave is done with its ring and its rows' bits
                if (hk == 0) s_state[w * kTaRows + hn] = make_float2(m_all, l_all);
                lds_sync();
                const float2 other = s_state[(w ^ R) * kTaRows + hn];
                const float top = fmaxf(m_all, other.x);
                const float mine = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_all - top);
                const float theirs = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(other.x - top);
                const float l = mine * l_all + theirs * other.y;
                const float factor = whole ? (l > 0.f || l != l ? 1.f / l : 0.f) : 1.f;
                const uint32_t out_lds = lds_addr(s_mem) + w * 4 * 4096 + le * 16;
                const uint32_t in_lds = lds_addr(s_mem) + (w ^ R) * 4 * 4096 + le * 16;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if (half > 0) lds_sync();
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if (j / 4 == st) continue;
                        hold(o[8 * half + j]);
#pragma unroll
                        for (int a = 0; a < 4; ++a) {
                            const v16f& x = o[8 * half + j];
                            *(LdsF32x4Out)(out_lds + ((j & 3) * 4 + a) * 1024) = f32x4{x[4 * a], x[4 * a + 1], x[4 * a + 2], x[4 * a + 3]} * mine;
                        }
                    }
                    lds_sync();
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if (j / 4 != st) continue;
                        hold(o[8 * half + j]);
                        v16f x = o[8 * half + j] * mine;
#pragma unroll
                        for (int a = 0; a < 4; ++a) {
                            const f32x4 add = *(LdsF32x4)(in_lds + ((j & 3) * 4 + a) * 1024);
#pragma unroll
                            for (int c = 0; c < 4; ++c) x[4 * a + c] += add[c];
                        }
                        put(8 * half + j, x, factor);
                    }
                }
                put_state(top, l);
            }
        }
        if (lane == 0) report(p.status, err);
        if (t0 == 0 && tid == 0) {  // which shares hold the item
            const int n = near, before_end = min(max(n, steps - n - 1), steps - 1);  // the last cut that leaves a step
            const int last = (item_pos + head + before_end) / quota;
            work.items[static_cast<int64_t>(b) * ta_tiles(p.max_nodes * p.heads, R) + rt] = make_int2(g, last - g + 1);
        }
    }
}

// Joins the parts of items that several shares hold. A workgroup of W waves takes 32 rows and U of the 64 units
// of 8 features at a time; its waves take every W-th part, and meet in LDS, from where a row's features are stored
// side by side. A lane holds four features of a row per unit, as the parts do. What bounds it is how many
// loads are under way and how many waves there are to start: few items have many parts, which go over more
// waves (2 requests of one token, 32 heads, up to 93000 rows: 43.5 us with 8, 49.5 with 4), many items have few and
// take more units per workgroup, and go on to the units `slices` further (U = 1 with W = 16 and no such loop took
// 3584 workgroups for 7 requests of 12 tokens x 20 heads, and 48 us instead of 29).
template <int R, int U, int W>
__global__ __launch_bounds__(W * 64) void tree_join_kernel(const KvipTreeAttnArgs p, int shares, int slices) {
    constexpr int kPitch = 65, kAtOnce = 16 / U;  // parts whose loads are issued together
    __shared__ f32x4 s_sums[W][U * kPitch];
    __shared__ float2 s_state[W][kTaRows];  // maximum and sum
    const int tiles = ta_tiles(p.max_nodes * p.heads, R);
    const int slice = blockIdx.x % slices, rg = blockIdx.x / slices % R, item = blockIdx.x / slices / R;
    const int b = item / tiles, rt = item % tiles;
    const TaWork<R> work(p.workspace, shares);
    int2 of = work.items[item];  // where the item has rows
    of.y = static_cast<unsigned>(of.x) < static_cast<unsigned>(shares) ? min(of.y, shares - of.x) : 0;
    uint32_t err = 0;
    const TaRequest req = ta_request(p, b, &err);
    const int rows = req.nodes * p.heads, first_row = (rt * R + rg) * kTaRows;
    if (first_row >= rows) return;
    if (of.y <= 1) return;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, n = lane & 31;
    auto part = [&](int k) { return (of.x + k) * 2 + (k == 0 ? 1 : 0); };  // of share of.x + k
    for (int unit = slice * U; unit < kBlocks * 4; unit += slices * U) {
        if (unit != slice * U) __syncthreads();  // the sums before are read
        float m = -INFINITY, l = 0.f;
        f32x4 v[U] = {};
        for (int k0 = w; k0 < of.y; k0 += W * kAtOnce) {
            float2 state[kAtOnce];
            f32x4 x[kAtOnce][U];
            float most = m;
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                const int k = k0 + i * W;
                state[i] = make_float2(-INFINITY, 0.f);
                if (k < of.y) {
                    state[i] = work.rows(part(k), rg)[n];
                    const f32x4* sums = work.group(part(k), rg) + unit * 64 + lane;
#pragma unroll
                    for (int u = 0; u < U; ++u) x[i][u] = __builtin_nontemporal_load(sums + u * 64);
                }
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) most = fmaxf(most, state[i].x);
            const float keep = most == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - most);
            l *= keep;
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] *= keep;
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                if (k0 + i * W >= of.y) break;
                const float weight = most == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(state[i].x - most);
                l += weight * state[i].y;
#pragma unroll
                for (int u = 0; u < U; ++u) v[u] += weight * x[i][u];
            }
            m = most;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) s_sums[w][u * kPitch + lane] = v[u];
        if (lane < kTaRows) s_state[w][n] = make_float2(m, l);
        __syncthreads();
        for (int i = threadIdx.x; i < kTaRows * U * 2; i += W * 64) {
            const int r = i / (U * 2), u = i / 2 % U, kg = i % 2;
            if (first_row + r >= rows) break;
            float most = -INFINITY, sum = 0.f;
#pragma unroll
            for (int k = 0; k < W; ++k) most = fmaxf(most, s_state[k][r].x);
            f32x4 out = {};
#pragma unroll
            for (int k = 0; k < W; ++k) {
                const float2 state = s_state[k][r];
                const float weight = most == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(state.x - most);
                sum += weight * state.y;
                out += weight * s_sums[k][u * kPitch + kg * kTaRows + r];
            }
            const int64_t out_row = static_cast<int64_t>(req.begin) * p.heads + first_row + r;
            ta_store(p, out_row * kValueDim + (unit + u) * 8 + kg * 4, out * (sum > 0.f || sum != sum ? 1.f / sum : 0.f));
            if (unit + u == 0 && kg == 0 && p.lse != nullptr) p.lse[out_row] = ta_lse(most, sum);
        }
    }
}

template <int R, int U, int W>
void launch_join(const KvipTreeAttnArgs& a, int shares, int groups, hipStream_t s) {
    int slices = kBlocks * 4 / U;
    while (slices > 1 && groups * slices * W > kJoinWaves) slices /= 2;
    hipLaunchKernelGGL((tree_join_kernel<R, U, W>), dim3(groups * slices), dim3(W * 64), 0, s, a, shares, slices);
}

template <int R>
void launch_tree(const KvipTreeAttnArgs& a, hipStream_t s) {
    const int shares = ta_shares(a.batch, a.heads, a.max_nodes, a.max_blocks);
    hipLaunchKernelGGL(tree_attention_kernel<R>, dim3(shares), dim3(kTaThreads), 0, s, a);
    // Few groups of 32 rows have many parts each, many have few (batches of 4 tokens x 16 heads on 2000-8000 rows with
    // 4 units and 8 waves / 4 and 4 / 8 and 4: 2 requests 29.1 / 29.4 / 32.5 us, 16 requests (32 groups) 40.8 / 41.1 /
    // 41.4, 64 (128 groups) 84.8 / 83.5 / 84.0; 1000 requests on 50-400 rows with 4 and 4 / 8 and 4: 149.6 / 145).
    const int groups = a.batch * ta_tiles(a.max_nodes * a.heads, R) * R;
    if (groups <= 32) launch_join<R, 4, 8>(a, shares, groups, s);
    else if (groups <= 128) launch_join<R, 4, 4>(a, shares, groups, s);
    else launch_join<R, 8, 4>(a, shares, groups, s);
}

}  // namespace
}  // namespace kvip

extern "C" uint64_t kvip_hip_tree_attention_workspace_bytes(int32_t batch, int32_t heads, int32_t max_nodes,
                                                            int32_t max_blocks) {
    if (batch < 1 || batch > KVIP_DRAFT_MAX_BATCH || heads < 1 || heads > 128 || max_nodes < 1 ||
        max_nodes > KVIP_DRAFT_MAX_NODES || max_blocks < 1 || max_blocks > (1 << 17) ||
        kvip::ta_most_steps(batch, heads, max_nodes, max_blocks) > 0x7FFFFFFF) {
        return 0;
    }
    const int r = kvip::ta_groups(heads, max_nodes), shares = kvip::ta_shares(batch, heads, max_nodes, max_blocks);
    return static_cast<uint64_t>(shares) * 2 * kvip::kTaRows * r * (kvip::kValueDim + 2) * sizeof(float) +
           static_cast<uint64_t>(batch) * kvip::ta_tiles(heads * max_nodes, r) * sizeof(int2);
}

extern "C" uint32_t kvip_hip_tree_attention(const KvipTreeAttnArgs* a, void* stream) {
    if (a == nullptr) return KVIP_ERR_INVALID;
    auto aligned = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15u) == 0; };
    const bool ok = a->query && a->kv_cache && a->block_table && a->seq_lens && a->cu_seqlens && a->output && a->workspace &&
                    aligned(a->query) && aligned(a->kv_cache) && aligned(a->output) && aligned(a->workspace) &&
                    a->batch >= 1 && a->batch <= KVIP_DRAFT_MAX_BATCH && a->heads >= 1 && a->heads <= 128 &&
                    a->max_nodes >= 1 && a->max_nodes <= KVIP_DRAFT_MAX_NODES && a->max_tokens >= 1 &&
                    a->max_tokens <= KVIP_DRAFT_MAX_TOKENS && a->max_blocks >= 1 && a->max_blocks <= (1 << 17) &&
                    a->num_blocks >= 1 && a->num_blocks < (1 << 24) && a->row_stride >= KVIP_KV_ROW_BYTES &&
                    a->row_stride <= (1 << 24) && a->row_stride % 16 == 0 && a->kv_block_stride % 16 == 0 &&
                    a->kv_block_stride >= static_cast<int64_t>(kvip::kBlockTokens) * a->row_stride &&
                    (a->output_dtype == KVIP_DTYPE_BF16 || a->output_dtype == KVIP_DTYPE_FP32) &&
                    a->scale - a->scale == 0.f &&  // finite
                    kvip::ta_most_steps(a->batch, a->heads, a->max_nodes, a->max_blocks) <= 0x7FFFFFFF;
    if (!ok) return KVIP_ERR_INVALID;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    switch (kvip::ta_groups(a->heads, a->max_nodes)) {
        case 2: kvip::launch_tree<2>(*a, s); break;
        default: kvip::launch_tree<4>(*a, s); break;
    }
    return static_cast<uint32_t>(hipGetLastError());
}
