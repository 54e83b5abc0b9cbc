// Attention of a request's step tokens (a tree of drafted tokens) over its paged KV rows; the rules
// stand in kvip_hip_draft.h. A row of the cache holds 512 fp8 e4m3 features with one fp32 scale per 128
// and 64 bf16 rotary features: key = [nope * scale, rope], value = nope * scale.
//
// The rows of the problem are a request's (step token, head) pairs, which all read the same cache rows.
// A workgroup of 4 waves takes R groups of 32 rows (R = 1, 2, 4) by 4 / R streams of 32-token tiles, a wave
// per group and stream. A wave keeps its 32 queries (36 fragments, 144 registers) and its 32 x 512
// accumulator (256 accumulation registers, one wave per SIMD has 512) and exchanges nothing until the
// streams are merged at the end:
//   - A tile stays as it is in the cache: direct-to-LDS loads put its fp8 bytes into a two-slot ring, the
//     next tile landing while this one is computed.
//   - Logits are computed transposed (tokens x rows): bf16 MFMA of the key bytes, converted as they are read
//     (exact), with the query; a scale group's dot products are summed on their own and added as
//     fma(group, scale, s) in fp32.
//   - So a lane holds one row's logits of 16 tokens: the softmax takes one lane swap per tile, and the
//     probabilities times the group's scale (rounded once to bf16) are the value product's operand
//     without leaving their registers, as the order of tokens along K is free. The value operand (8
//     tokens of one feature per lane) comes from the token-major tile by transposing LDS reads.
//   - The running maximum is raised lazily, when a tile exceeds it by kTaMargin.
//
// The (request, row tile, token steps) are laid out in one line and cut into equal shares, one per
// workgroup, so that ragged batches keep every CU busy; what a share has of an item that others
// share goes to the workspace, and a second launch joins the parts.
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
constexpr int kKeyDim = 576;                // 512 nope + 64 rope
constexpr int kValueDim = 512;
constexpr int kScaleGroups = 4;
constexpr int kBlocks = kValueDim / 32;     // accumulator blocks of 32 features
constexpr int kTaGroups = 256;              // shares: one workgroup per CU
constexpr int kMinSteps = 4;                // steps of a share, at least
constexpr int kJoinRows = 8;                // rows per workgroup of the joining launch
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f;
constexpr float kTaMargin = 8.0f * kLog2e;

constexpr int kNopeSlot = kTaTile * kValueDim;
constexpr int kRopeSlot = kTaTile * 128;
constexpr int kScaleSlot = kScaleGroups * kTaTile * 4;

// LDS of a workgroup with R row groups: per stream two slots of nope bytes, one (R = 1: LDS has no room
// for two) or two of rope, two of scales [group][token]; then the work line's prefix sums. The merge of the
// streams takes the front (8 blocks of 4 KB per wave).
template <int R>
struct TaLds {
    static constexpr int kStreams = kTaWaves / R;
    static constexpr int kRopeSlots = R == 1 ? 1 : 2;
    static constexpr int kRope = kStreams * 2 * kNopeSlot;
    static constexpr int kScale = kRope + kStreams * kRopeSlots * kRopeSlot;
    static constexpr int kFront = kScale + kStreams * 2 * kScaleSlot;
    static constexpr int kMerge = kStreams == 1 ? 0 : kTaWaves * 8 * 4096;
    static constexpr int kState = kFront > kMerge ? kFront : kMerge;  // [wave][row] maximum and sum
    static constexpr int kLine = kState + kTaWaves * kTaRows * 8;
    static constexpr int kBytes = kLine + (KVIP_DRAFT_MAX_BATCH + 1) * 8 + 64;
    static_assert(kBytes <= 160 * 1024, "LDS of a CU");
};

__host__ __device__ inline int ta_groups(int heads, int nodes) {  // R
    const int rows = heads * nodes;
    return rows <= kTaRows ? 1 : rows <= 2 * kTaRows ? 2 : 4;
}

__host__ __device__ inline int ta_tiles(int rows, int r) { return (rows + kTaRows * r - 1) / (kTaRows * r); }

// Shares of a launch: no more than the longest contexts could fill.
__host__ __device__ inline int ta_shares(int batch, int heads, int nodes, int max_blocks) {
    const int r = ta_groups(heads, nodes), streams = kTaWaves / r;
    const int64_t steps = (static_cast<int64_t>(max_blocks) * kBlockTokens + kTaTile * streams - 1) / (kTaTile * streams);
    const int64_t most = (steps * batch * ta_tiles(heads * nodes, r) + kMinSteps - 1) / kMinSteps;
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

// acc += a0 b0 + a1 b1 with the accumulator in accumulation registers. The compiler, left to choose, moves
// parts of the 256 accumulators between the two halves of the register file in every tile. It does not
// see what this block holds, so the block waits itself: two states between a vector write of an operand
// and its reading. Nothing reads an accumulator within a tile of its last product (accumulators_done).
KVIP_DEVICE void mma_pair(v16f& acc, bf16x8 a0, bf16x8 b0, bf16x8 a1, bf16x8 b1) {
    asm volatile(
        "s_nop 1\n\t"
        "v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0\n\t"
        "v_mfma_f32_32x32x16_bf16 %0, %3, %4, %0"
        : "+a"(acc) : "v"(a0), "v"(b0), "v"(a1), "v"(b1));
}

// The products of mma_pair are in the accumulators (18 states after the last are enough).
KVIP_DEVICE void accumulators_done(v16f (&o)[kBlocks]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        asm volatile("s_nop 15\n\ts_nop 7"
                     : "+a"(o[8 * h]), "+a"(o[8 * h + 1]), "+a"(o[8 * h + 2]), "+a"(o[8 * h + 3]), "+a"(o[8 * h + 4]),
                       "+a"(o[8 * h + 5]), "+a"(o[8 * h + 6]), "+a"(o[8 * h + 7]));
    }
}

// Where the workspace holds what: per share two parts (its first item's, where others began it, and its
// last one's, where others go on) of 32 R rows x 512 sums, their (maximum, sum) pairs, then per item the
// first share and the number of shares.
template <int R>
struct TaWork {
    float* sums;
    float2* state;
    int2* items;
    KVIP_DEVICE TaWork(void* base, int shares) {
        constexpr int kRowsOf = kTaRows * R;
        sums = static_cast<float*>(base);
        state = reinterpret_cast<float2*>(sums + static_cast<size_t>(shares) * 2 * kRowsOf * kValueDim);
        items = reinterpret_cast<int2*>(state + static_cast<size_t>(shares) * 2 * kRowsOf);
    }
};

// A request as the kernel takes it.
struct TaRequest {
    int begin;   // first row of the step
    int nodes;   // its step tokens (at most max_nodes)
    int past;    // position of step token 0 (below 0 where the length is too short)
    int length;  // cache rows
};

KVIP_DEVICE TaRequest ta_request(const KvipTreeAttnArgs& p, int b, uint32_t* err) {
    TaRequest q;
    q.begin = min(max(p.cu_seqlens[b], 0), p.max_tokens);
    const int all = min(max(p.cu_seqlens[b + 1], q.begin), p.max_tokens) - q.begin;
    const int given = p.seq_lens[b];
    q.nodes = min(all, p.max_nodes);
    q.length = min(max(given, 0), p.max_blocks * kBlockTokens);
    q.past = q.length - all;
    if (given != q.length || all != q.nodes || (all > 0 && q.past < 0)) *err |= KVIP_STATUS_BAD_LENGTH;
    return q;
}

// Steps of an item: at least one, so that rows without any token get their zeros.
template <int R>
KVIP_DEVICE int ta_steps(int length) {
    constexpr int kTokens = kTaTile * (kTaWaves / R);
    return max((length + kTokens - 1) / kTokens, 1);
}

template <int R>
__global__ __launch_bounds__(kTaThreads, 1) void tree_attention_kernel(const KvipTreeAttnArgs p) {
    typedef TaLds<R> L;
    constexpr int kStreams = L::kStreams;
    __shared__ __align__(1024) uint8_t s_mem[L::kBytes];
    int64_t* s_line = reinterpret_cast<int64_t*>(s_mem + L::kLine);  // steps before each request
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rg = w % R, st = w / R;
    const int n = lane & 31, kg = lane >> 5;

    // The line of work: 4 requests per thread, running sums in 64 bits.
    {
        constexpr int kPer = KVIP_DRAFT_MAX_BATCH / kTaThreads;
        int64_t* s_sum = s_line + KVIP_DRAFT_MAX_BATCH + 1;
        int64_t steps[kPer], sum = 0;
        uint32_t err = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int b = tid * kPer + i;
            steps[i] = 0;
            if (b < p.batch) {
                const TaRequest q = ta_request(p, b, &err);
                steps[i] = static_cast<int64_t>(ta_tiles(q.nodes * p.heads, R)) * ta_steps<R>(q.length);
            }
            sum += steps[i];
        }
        if (blockIdx.x == 0) report(p.status, err);
        int64_t run = sum;
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t lo = static_cast<uint32_t>(__shfl_up(static_cast<int>(run), d));
            const uint32_t hi = static_cast<uint32_t>(__shfl_up(static_cast<int>(run >> 32), d));
            if (lane >= d) run += static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
        }
        if (lane == 63) s_sum[w] = run;
        __syncthreads();
        int64_t before = run - sum;
        for (int v = 0; v < w; ++v) before += s_sum[v];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int b = tid * kPer + i;
            if (b <= p.batch) s_line[b] = before;
            before += steps[i];
            if (b == p.batch - 1) s_line[p.batch] = before;
        }
        __syncthreads();
    }
    const int64_t total = s_line[p.batch];
    const int shares = gridDim.x;
    const int64_t even = (total + shares - 1) / shares, quota = even < kMinSteps ? kMinSteps : even;
    // Neighbouring shares, which read the same cache rows where an item or a request spans them, on one
    // XCD (workgroups are dealt round the 8).
    const int per_xcd = shares / 8;
    const int g = static_cast<int>(blockIdx.x) < per_xcd * 8 ? static_cast<int>(blockIdx.x % 8) * per_xcd + blockIdx.x / 8
                                                             : blockIdx.x;
    int64_t pos = min(g * quota, total);
    const int64_t end = min(pos + quota, total);
    const TaWork<R> work(p.workspace, shares);

    uint8_t* ring = s_mem + st * 2 * kNopeSlot;
    const uint32_t ring_lds = lds_addr(ring);
    const uint32_t rope_lds = lds_addr(s_mem + L::kRope + st * L::kRopeSlots * kRopeSlot);
    const uint32_t scales_lds = lds_addr(s_mem + L::kScale + st * 2 * kScaleSlot);
    const float scale2 = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(p.scale * kLog2e)));
    const int64_t row_stride = p.row_stride;

    while (pos < end) {
        // The item at `pos`: request b, row tile rt, steps t0 .. t1 of its `steps`.
        int b = 0;
        {
            int lo = 0, hi = p.batch - 1;  // the last request that starts at or before pos
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (s_line[mid] <= pos) lo = mid;
                else hi = mid - 1;
            }
            b = __builtin_amdgcn_readfirstlane(lo);
        }
        uint32_t err = 0;
        const TaRequest req = ta_request(p, b, &err);
        err = 0;
        const int steps = ta_steps<R>(req.length);
        const int64_t within = pos - s_line[b];
        const int rt = __builtin_amdgcn_readfirstlane(static_cast<int>(within / steps));
        const int t0 = __builtin_amdgcn_readfirstlane(static_cast<int>(within % steps));
        const int t1 = __builtin_amdgcn_readfirstlane(static_cast<int>(min(static_cast<int64_t>(steps), t0 + (end - pos))));
        const int64_t item_pos = pos - t0;
        pos += t1 - t0;
        const bool whole = t0 == 0 && t1 == steps;
        const int rows = req.nodes * p.heads;
        const int row = rt * kTaRows * R + rg * kTaRows + n;
        const bool busy = rt * kTaRows * R + rg * kTaRows < rows;  // uniform: the wave's group has rows
        const int32_t* table = p.block_table + static_cast<int64_t>(b) * p.max_blocks;

        // Page of the wave's tile of step k (-1: none of its tokens is there).
        auto page_of = [&](int k) {
            const int t = k * kStreams + st;
            int page = -1;
            if (k < t1 && t * kTaTile < req.length) {
                page = table[t / (kBlockTokens / kTaTile)];
                if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.num_blocks)) {
                    err |= KVIP_STATUS_BAD_BLOCK;
                    page = -1;
                }
            }
            return page;
        };
        // First byte of the tile's first row.
        auto tile_base = [&](int k, int page) {
            const int t = k * kStreams + st;
            return p.kv_cache + page * p.kv_block_stride + (t % (kBlockTokens / kTaTile)) * kTaTile * row_stride;
        };
        // This wave's share (1 / R) of the loads of a tile's nope bytes and scales into slot `slot`. LDS row t
        // holds piece s ^ swz(t) at place s. Tokens past the length get zeros: their probabilities are
        // zero, and zero times a stray NaN would not be.
        auto load_nope = [&](int k, int page, int slot) {
            const int ln = fresh(lane), up = ln >> 5;
            const int live = min(req.length - (k * kStreams + st) * kTaTile, kTaTile);
            constexpr int kLoads = 16 / R;  // of tokens 2 v and 2 v + 1 each
            const uint8_t* base = tile_base(k, page) + up * row_stride;
            const int from = ((ln & 31) ^ ta_swz(up)) * 16;
            const uint32_t dst = ring_lds + slot * kNopeSlot;
#pragma unroll
            for (int x = 0; x < kLoads; ++x) {
                const int v = rg * kLoads + x;
                const uint8_t* src = base + 2 * v * row_stride + (from ^ (ta_swz(2 * v) * 16));
                if (live == kTaTile || 2 * v + up < live) {
                    dma16(src, dst + v * 1024);
                } else {
                    *(__attribute__((address_space(3))) v4i*)(dst + v * 1024 + ln * 16) = v4i{0, 0, 0, 0};
                }
            }
            // Scales, as [group][token]: groups 2 v and 2 v + 1 per load, v = 0 and 1.
            const uint8_t* src = tile_base(k, page) + (ln & 31) * row_stride + 640 + 4 * up;
            const uint32_t sc = scales_lds + slot * kScaleSlot;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                if (R > 1 && v != rg) continue;
                if (live == kTaTile || (ln & 31) < live) dma4(src + 8 * v, sc + v * 256);
                else *(__attribute__((address_space(3))) float*)(sc + v * 256 + ln * 4) = 0.f;
            }
        };
        // And of its rope features: LDS row t (128 bytes) holds piece s ^ (t / 2 % 8) at place s. Tokens past the
        // length keep stale bytes: their logits are replaced.
        auto load_rope = [&](int k, int page, int slot) {
            const int ln = fresh(lane);
            const int live = min(req.length - (k * kStreams + st) * kTaTile, kTaTile);
            constexpr int kLoads = 4 / R;  // of tokens 8 v .. 8 v + 7 each
#pragma unroll
            for (int x = 0; x < kLoads; ++x) {
                const int v = rg * kLoads + x, token = 8 * v + (ln >> 3);
                const int piece = (ln & 7) ^ ((token >> 1) & 7);
                if (token < live) {
                    dma16(tile_base(k, page) + token * row_stride + kValueDim + piece * 16,
                          rope_lds + (L::kRopeSlots == 1 ? 0 : slot * kRopeSlot) + v * 1024);
                }
            }
        };
        // Every load and LDS access of this wave is done, and (waves sharing a stream) of all waves.
        auto settle = [&] {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");
            if constexpr (R > 1) __builtin_amdgcn_s_barrier();
            asm volatile("" : : : "memory");
        };

        __syncthreads();  // the LDS of the item before is free
        int page = page_of(t0);
        if (page >= 0) {
            load_nope(t0, page, 0);
            load_rope(t0, page, 0);
        }
        int page_next = page_of(t0 + 1);

        // Queries of the wave's rows (rows past the last read it again; their outputs are not written). Fragment
        // (group g, j, x): features 16 (8 g + 2 j + kg) + 8 x .. + 7, the half x of the key piece that the lane
        // reads; the last four: rope features 16 i + 8 kg .. + 7.
        bf16x8 qf[36];
        uint64_t seen;
        {
            const int at = min(row, rows - 1), node = at / p.heads;
            const uint16_t* q = p.query + (static_cast<int64_t>(req.begin) * p.heads + at) * kKeyDim;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                qf[i] = *reinterpret_cast<const bf16x8*>(q + (i >> 1) * 32 + kg * 16 + (i & 1) * 8);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) qf[32 + i] = *reinterpret_cast<const bf16x8*>(q + kValueDim + i * 16 + kg * 8);
            seen = p.visible != nullptr ? static_cast<uint64_t>(p.visible[req.begin + node]) : ~0ull >> (63 - node);
        }
        v16f o[kBlocks];
#pragma unroll
        for (int f = 0; f < kBlocks; ++f) {
#pragma unroll
            for (int i = 0; i < 16; ++i) o[f][i] = 0.f;
        }
        float m_run = -INFINITY;  // reference maximum of the row, log2 units
        float l_sum = 0.f;        // this lane's share of its probability sum
        // Waited for here: the tile loop would wait for them each time round, and so for its own loads.
#pragma unroll
        for (int i = 0; i < 36; ++i) asm volatile("" : "+v"(qf[i]));

        int slot = 0;
#pragma unroll 1
        for (int k = t0; k < t1; ++k, slot ^= 1) {
            settle();  // the tile has landed; the other slot is free
            const int ahead = page_next;
            page_next = page_of(k + 2);
            if (ahead >= 0) {
                load_nope(k + 1, ahead, slot ^ 1);
                if (L::kRopeSlots == 2) load_rope(k + 1, ahead, slot ^ 1);
            }
            const int ln = fresh(lane), tn = ln & 31, tk = ln >> 5;
            const uint32_t ro = rope_lds + (L::kRopeSlots == 1 ? 0 : slot * kRopeSlot) + tn * 128;
            const uint32_t ko = ring_lds + slot * kNopeSlot + tn * kValueDim + ((tk ^ ta_swz(tn)) << 4);
            const uint32_t sl = scales_lds + slot * kScaleSlot + 16 * tk;  // scales of tokens 8 a + 4 kg .. + 3
            const int y = (ln & 15) >> 1, vt = 8 * (y >> 2) + 4 * tk + (y & 3);
            const uint32_t vo = ring_lds + slot * kNopeSlot + vt * kValueDim + ((((ln >> 4) & 1) ^ ta_swz(vt)) << 4) + 8 * (ln & 1);

            v16f s;
            if (busy && page >= 0) {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const v4i x = *(LdsV4i)(ro + (((2 * i + tk) ^ ((tn >> 1) & 7)) << 4));
                    s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), qf[32 + i], s, 0, 0, 0);
                }
            }
            if (L::kRopeSlots == 1 && ahead >= 0) {  // the single rope slot has been read
                asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
                load_rope(k + 1, ahead, 0);
            }
            const int first = (k * kStreams + st) * kTaTile;  // position of the tile's first token
            // A step with step tokens or the end of the context in it (the same for the workgroup's waves). What
            // a row does not see must not reach it, and zero times a NaN would: tokens with a NaN feature or a
            // scale that is not finite are found and zeroed in LDS, and rows that do see one become NaN as a whole
            // (their logit is none).
            uint32_t sees = 0xFFFFu;  // bit i: the row sees the token of register i
            if ((k + 1) * kStreams * kTaTile > req.past) {
                uint32_t nan = 0;
                const uint32_t at = ring_lds + slot * kNopeSlot + tn * kValueDim;
                const uint32_t sc = scales_lds + slot * kScaleSlot + tk * 2 * kTaTile * 4 + tn * 4;
                if (page >= 0) {
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
                }
                const uint64_t found = __ballot(nan != 0);
                const uint32_t bad = static_cast<uint32_t>(found | found >> 32);
                if constexpr (R > 1) {  // the waves of the stream have all looked
                    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
                    __builtin_amdgcn_s_barrier();
                    asm volatile("" : : : "memory");
                }
                if (bad >> tn & 1) {
#pragma unroll 1
                    for (int i = 0; i < 16; ++i) {
                        *(__attribute__((address_space(3))) v4i*)(at + (16 * tk + i) * 16) = v4i{0, 0, 0, 0};
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) *(__attribute__((address_space(3))) float*)(sc + i * kTaTile * 4) = 0.f;
                }
                sees = 0;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int token = 8 * (i >> 2) + 4 * tk + (i & 3), rel = first + token - req.past;
                    const bool in = rel < 0 || (rel < KVIP_DRAFT_MAX_NODES && rel < req.length - req.past &&
                                                (seen >> (rel & 63) & 1) != 0);
                    sees |= in ? 1u << i : 0u;
                    if (in && (bad >> token & 1)) l_sum = NAN;
                }
            }
            if (busy && page >= 0) {
#pragma unroll
                for (int gr = 0; gr < kScaleGroups; ++gr) {
                    v16f dot;
#pragma unroll
                    for (int i = 0; i < 16; ++i) dot[i] = 0.f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const v4i x = *(LdsV4i)(ko ^ ((8 * gr + 2 * j) * 16));
                        dot = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fp8x8_to_bf16(x[0], x[1]), qf[8 * gr + 2 * j], dot, 0, 0, 0);
                        dot = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fp8x8_to_bf16(x[2], x[3]), qf[8 * gr + 2 * j + 1], dot, 0, 0, 0);
                    }
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        const f32x4 s4 = *(LdsF32x4)(sl + (gr * kTaTile + 8 * a) * 4);
#pragma unroll
                        for (int c = 0; c < 4; ++c) s[4 * a + c] = fmaf(dot[4 * a + c], s4[c], s[4 * a + c]);
                    }
                }
                // Softmax: pr = 2^(logit - m), the logits of tokens that the row does not see at -inf.
                float pr[16], mx = -INFINITY;
#pragma unroll
                for (int i = 0; i < 16; ++i) pr[i] = s[i] * scale2;
                if (first + kTaTile > req.past) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        if (!(sees >> i & 1)) pr[i] = -INFINITY;
                    }
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) mx = fmaxf(mx, pr[i]);
                mx = half_max(mx);
                const bool raise = mx > m_run + kTaMargin;  // also the first finite maximum
                if (__ballot(raise) != 0ull) {
                    const float m_new = raise ? mx : m_run;
                    const float alpha = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - m_new);
                    const float a = raise ? alpha : 1.f;
                    l_sum *= a;
#pragma unroll
                    for (int f = 0; f < kBlocks; ++f) {
                        asm volatile("" : "+a"(o[f]));  // read here, not in every tile
                        o[f] *= a;
                        asm volatile("" : "+a"(o[f]));
                    }
                    m_run = m_new;
                }
                const float bias = m_run == -INFINITY ? 0.f : -m_run;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    pr[i] = __builtin_amdgcn_exp2f(pr[i] + bias);
                    l_sum += pr[i];
                }
                // Value product [features, rows].
#pragma unroll
                for (int gr = 0; gr < kScaleGroups; ++gr) {
                    v4i packed[2];
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        const f32x4 s4 = *(LdsF32x4)(sl + (gr * kTaTile + 8 * a) * 4);
                        packed[a >> 1][2 * (a & 1)] = static_cast<int>(pack_bf16(pr[4 * a] * s4[0], pr[4 * a + 1] * s4[1]));
                        packed[a >> 1][2 * (a & 1) + 1] = static_cast<int>(pack_bf16(pr[4 * a + 2] * s4[2], pr[4 * a + 3] * s4[3]));
                    }
                    const bf16x8 p0 = __builtin_bit_cast(bf16x8, packed[0]), p1 = __builtin_bit_cast(bf16x8, packed[1]);
#pragma unroll
                    for (int f = 4 * gr; f < 4 * gr + 4; ++f) {
                        const i32x2 v0 = __builtin_amdgcn_ds_read_tr8_b64_v2i32((LdsI32x2)(vo ^ (f * 32)));
                        const i32x2 v1 = __builtin_amdgcn_ds_read_tr8_b64_v2i32((LdsI32x2)((vo ^ (f * 32)) + 16 * kValueDim));
                        mma_pair(o[f], fp8x8_to_bf16(v0[0], v0[1]), p0, fp8x8_to_bf16(v1[0], v1[1]), p1);
                    }
                }
            }
            page = ahead;
        }
        accumulators_done(o);
        if (lane == 0) report(p.status, err);

        // Merge of the streams: with the maximum M over them, sums = sum_w 2^(m_w - M) o_w and l likewise. A wave
        // sums 16 / streams of the blocks, from halves of 8 blocks that the others put into LDS.
        const float l_all = half_sum(l_sum);
        float m = m_run, l = l_all, mine = 1.f;
        float2* s_state = reinterpret_cast<float2*>(s_mem + L::kState);
        if constexpr (kStreams > 1) {
            if (kg == 0) s_state[w * kTaRows + n] = make_float2(m_run, l_all);
            __syncthreads();  // and every wave is done with its ring
            m = -INFINITY;
#pragma unroll
            for (int v = 0; v < kStreams; ++v) m = fmaxf(m, s_state[(v * R + rg) * kTaRows + n].x);
            l = 0.f;
#pragma unroll
            for (int v = 0; v < kStreams; ++v) {
                const float2 sv = s_state[(v * R + rg) * kTaRows + n];
                const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sv.x - m);
                l += f * sv.y;
                if (v == st) mine = f;
            }
        }
        const int64_t out_row = static_cast<int64_t>(req.begin) * p.heads + row;
        // A whole item's rows are final; else the sums and their state go to the share's part 0 (others began
        // the item) or 1.
        const float factor = whole ? (l > 0.f || l != l ? 1.f / l : 0.f) : 1.f;
        const size_t slot_row = (static_cast<size_t>(g) * 2 + (t0 == 0 ? 1 : 0)) * kTaRows * R + rg * kTaRows + n;
        auto put = [&](int f, const v16f& x) {
            if (row >= rows) return;
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const int feature = 32 * f + 8 * a + 4 * kg;
                const f32x4 v = f32x4{x[4 * a], x[4 * a + 1], x[4 * a + 2], x[4 * a + 3]} * factor;
                if (!whole) {
                    *reinterpret_cast<f32x4*>(work.sums + slot_row * kValueDim + feature) = v;
                } else if (p.output_dtype == KVIP_DTYPE_FP32) {
                    *reinterpret_cast<f32x4*>(static_cast<float*>(p.output) + out_row * kValueDim + feature) = v;
                } else {
                    *reinterpret_cast<bf16x4*>(static_cast<__bf16*>(p.output) + out_row * kValueDim + feature) =
                        __builtin_convertvector(v, bf16x4);
                }
            }
        };
        if constexpr (kStreams == 1) {
            if (busy) {
#pragma unroll
                for (int f = 0; f < kBlocks; ++f) put(f, o[f]);
            }
        } else {
            constexpr int kOwn = 8 / kStreams;  // blocks of a half that a wave sums
            const uint32_t buffer = lds_addr(s_mem);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                if (half > 0) __syncthreads();
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (j / kOwn == st || !busy) continue;
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        const v16f& x = o[8 * half + j];
                        *(LdsF32x4Out)(buffer + ((w * 8 + j) * 4 + a) * 1024 + lane * 16) =
                            f32x4{x[4 * a], x[4 * a + 1], x[4 * a + 2], x[4 * a + 3]} * mine;
                    }
                }
                __syncthreads();
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (j / kOwn != st || !busy) continue;
                    v16f x = o[8 * half + j] * mine;
#pragma unroll
                    for (int d = 1; d < kStreams; ++d) {
                        const int v = (st + d) % kStreams * R + rg;
#pragma unroll
                        for (int a = 0; a < 4; ++a) {
                            const f32x4 add = *(LdsF32x4)(buffer + ((v * 8 + j) * 4 + a) * 1024 + lane * 16);
#pragma unroll
                            for (int c = 0; c < 4; ++c) x[4 * a + c] += add[c];
                        }
                    }
                    put(8 * half + j, x);
                }
            }
        }
        if (st == 0 && kg == 0 && row < rows) {
            if (!whole) {
                work.state[slot_row] = make_float2(m, l);
            } else if (p.lse != nullptr) {
                p.lse[out_row] = l > 0.f || l != l ? (m + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
            }
        }
        if (t0 == 0 && tid == 0) {  // which shares hold the item
            const int last = static_cast<int>((item_pos + steps - 1) / quota);
            work.items[static_cast<int64_t>(b) * ta_tiles(p.max_nodes * p.heads, R) + rt] = make_int2(g, last - g + 1);
        }
    }
}

// Joins the parts of items that several shares hold: 8 rows per workgroup, 128 threads of 4 features per
// row and pass.
template <int R>
__global__ __launch_bounds__(kTaThreads) void tree_join_kernel(const KvipTreeAttnArgs p, int shares) {
    constexpr int kPer = kTaRows * R / kJoinRows;
    const int tiles = ta_tiles(p.max_nodes * p.heads, R);
    const int item = blockIdx.x / kPer, b = item / tiles, rt = item % tiles;
    uint32_t err = 0;
    const TaRequest req = ta_request(p, b, &err);
    const int rows = req.nodes * p.heads;
    const int local = static_cast<int>(blockIdx.x % kPer) * kJoinRows;
    if (rt * kTaRows * R + local >= rows) return;
    const TaWork<R> work(p.workspace, shares);
    const int2 of = work.items[item];
    if (of.y <= 1) return;
    const int f = (threadIdx.x & 127) * 4;
#pragma unroll 1
    for (int i = threadIdx.x >> 7; i < kJoinRows; i += 2) {
        const int row = rt * kTaRows * R + local + i;
        if (row >= rows) return;
        auto at = [&](int k) {  // the row of share of.x + k's part
            return (static_cast<size_t>(of.x + k) * 2 + (k == 0 ? 1 : 0)) * kTaRows * R + local + i;
        };
        float m = -INFINITY;
        for (int k = 0; k < of.y; ++k) m = fmaxf(m, work.state[at(k)].x);
        float l = 0.f;
        f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int k = 0; k < of.y; ++k) {
            const float2 sk = work.state[at(k)];
            const f32x4 x = *reinterpret_cast<const f32x4*>(work.sums + at(k) * kValueDim + f);
            const float wgt = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sk.x - m);
            l += wgt * sk.y;
            v += wgt * x;
        }
        v *= l > 0.f || l != l ? 1.f / l : 0.f;
        const int64_t out_row = static_cast<int64_t>(req.begin) * p.heads + row;
        if (p.output_dtype == KVIP_DTYPE_FP32) {
            *reinterpret_cast<f32x4*>(static_cast<float*>(p.output) + out_row * kValueDim + f) = v;
        } else {
            *reinterpret_cast<bf16x4*>(static_cast<__bf16*>(p.output) + out_row * kValueDim + f) =
                __builtin_convertvector(v, bf16x4);
        }
        if (f == 0 && p.lse != nullptr) {
            p.lse[out_row] = l > 0.f || l != l ? (m + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
        }
    }
}

template <int R>
void launch_tree(const KvipTreeAttnArgs& a, hipStream_t s) {
    const int shares = ta_shares(a.batch, a.heads, a.max_nodes, a.max_blocks);
    hipLaunchKernelGGL(tree_attention_kernel<R>, dim3(shares), dim3(kTaThreads), 0, s, a);
    const int items = a.batch * ta_tiles(a.max_nodes * a.heads, R);
    hipLaunchKernelGGL(tree_join_kernel<R>, dim3(items * (kTaRows * R / kJoinRows)), dim3(kTaThreads), 0, s, a, shares);
}

}  // namespace
}  // namespace kvip

extern "C" uint64_t kvip_hip_tree_attention_workspace_bytes(int32_t batch, int32_t heads, int32_t max_nodes,
                                                            int32_t max_blocks) {
    if (batch < 1 || batch > KVIP_DRAFT_MAX_BATCH || heads < 1 || heads > 128 || max_nodes < 1 ||
        max_nodes > KVIP_DRAFT_MAX_NODES || max_blocks < 1 || max_blocks > (1 << 17)) {
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
                    a->row_stride % 16 == 0 && a->kv_block_stride % 16 == 0 &&
                    a->kv_block_stride >= static_cast<int64_t>(kvip::kBlockTokens) * a->row_stride &&
                    (a->output_dtype == KVIP_DTYPE_BF16 || a->output_dtype == KVIP_DTYPE_FP32);
    if (!ok) return KVIP_ERR_INVALID;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    switch (kvip::ta_groups(a->heads, a->max_nodes)) {
        case 1: kvip::launch_tree<1>(*a, s); break;
        case 2: kvip::launch_tree<2>(*a, s); break;
        default: kvip::launch_tree<4>(*a, s); break;
    }
    return static_cast<uint32_t>(hipGetLastError());
}
