// Attention of chunks of new tokens over the paged KV rows (kvip_hip_prompt.h).
//
// The rows of the problem are a request's (chunk token, head) pairs. There are many per cached row, so a cached row
// is read by many workgroups, and converting its fp8 features in every one of them costs more than the products
// (attention of a few step tokens over the same rows spends 10 vector instructions per MFMA that way and reaches 795
// TFLOP/s). So the rows are laid out once, as fp16, in the order in which the tile loop wants them in LDS (expand): a
// tile of 32 rows is an image of 72 pieces x 32 rows x 16 bytes that direct-to-LDS loads copy as it stands.
//
// fp16 and not bf16, as a feature is an fp8 number times a 32-bit scale and a probability any number: in bf16 the
// roundings of keys, values and probabilities each add 0.0012 to an output's 0.0017 of error on 1030 cached rows (less on
// more rows, which average them); in fp16 nothing is left of them. What fp16 lacks is range, so an image stands under the
// exponent of its largest feature, each row under its own where the rows are far apart (what a token sees must not depend
// on what it does not); the sums of a row of the problem stand under the largest exponent of the cached rows that
// it has seen, and probabilities are lifted to the top of the range. bf16 was 10 % faster (6.83 instead of 7.63
// ms on the second of the cases below), the card at 1.8 GHz under either.
//
// A workgroup of 4 waves takes 128 rows of the problem, 32 per wave; a wave keeps its queries (144 registers) and its
// 32 x 512 sums (the 256 accumulation registers; one wave per SIMD has 512 in all). Logits are computed transposed (cached
// rows x rows of the problem), so that a lane holds one row's logits of 16 cached rows: the softmax takes one lane swap
// per tile, and the probabilities are the value product's operand in the lane that has them, as the order of cached
// rows along K is free. The value operand is read transposed from the same image. The running maximum is raised
// lazily, when a tile exceeds it by kCaMargin.
// One wave per SIMD hides nothing by itself, so the loop is one stretch of 68 MFMAs with everything else in between: the
// logits of tile t + 1, then the values of tile t with the softmax of tile t + 1 beside them. Operands are read from
// LDS four products ahead, across the borders of the two; the barrier for the tile after next stands where a tile's last
// reads are done.
//
// Few row tiles over long contexts are cut along the context into segments, whose parts a third launch joins: outputs of the
// segment's rows alone with their sums, as weighted sums of large values would pass 32 bits. Requests are taken the longest
// first.
//
// What bounds it. 2048 tokens x 128 heads on 8192 rows: 3.4-3.5 ms, 1170-1200 TFLOP/s, and 4096 tokens x 16 heads on 65536
// rows: 7.4-7.7 ms, 1170-1220 TFLOP/s, of the 1360 of a large fp16 product (on another card 4.0 and 8.7 ms): an MFMA is under
// way in 64 % of the cycles, at 1.78 GHz. The LDS is as busy, since every MFMA takes 1 KB from it, which four SIMDs without a pause
// would make all of its 128 bytes a cycle; without half of these reads the second case took 6 % less (wrong results, for
// the time alone). The clock is the card's answer to its power, and waves wait in 26 % of their cycles. Laying the rows out takes 11
// and 26 us. 12 requests of 1-700 tokens x 16 heads on up to 16000 rows: 1.14-1.17 ms, 1030 TFLOP/s, as the last workgroup
// ends 10 % after the mean CU's work. 130 tokens x 16 heads on 1030 rows: 6.5 + 22 + 8.5 us, chains of latencies (plan, images,
// queries to fp16, five tiles, parts, join).
// What it does not do: contexts are cut only where the whole batch has at most 512 row tiles, so that one long context among
// more of them is walked by its workgroups alone, some 1.9 us for every 32 rows; and few-row requests beside others
// are laid out like these (see ca_few).
// Dropped after measuring: operands eight products ahead and two accumulators for the logits in turn (both +-0 %), other
// prices of a part in the plan (+-2 % on small calls).
#include <type_traits>
#include <utility>

#include "kvip_hip_prompt.h"
#include "lane_groups.h"
#include "lds_async.h"

namespace kvip {
namespace {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4* LdsS16x4;

constexpr int kCaThreads = 256;
constexpr int kCaWaves = 4;
constexpr int kCaRows = 32;                       // rows of the problem per wave (MFMA N)
constexpr int kCaTileRows = kCaRows * kCaWaves;   // ... per workgroup
constexpr int kCaTile = 32;                       // cached rows of a tile (MFMA M of the logits)
constexpr int kCaKey = 576, kCaValue = 512;
constexpr int kCaBlocks = kCaValue / 32;          // accumulator blocks of 32 features
constexpr int kCaFrags = kCaKey / 16;             // MFMAs of a tile's logits
constexpr int kCaPieces = kCaKey / 8;
constexpr int kCaImage = kCaPieces * kCaTile * 16;
constexpr int kCaSlots = 4;                       // images in LDS
constexpr int kCaLoads = kCaImage / 1024 / kCaWaves;
constexpr int kCaUnits = 1024;                    // workgroups of a launch whose row tiles are cut, at most
constexpr int kCaCutTiles = 512;                  // row tiles that are cut, at most
constexpr int kCaMostCuts = 32;
constexpr int kCaPartSteps = 10;                  // what storing and joining a part costs, in tiles
constexpr int kCaCus = 256;
constexpr float kCaLog2e = 1.44269504088896341f;
constexpr float kCaLargest = 3.402823466e38f;
constexpr float kCaLn2 = 0.693147180559945309f;
constexpr float kCaMargin = 3.0f * kCaLog2e;
constexpr int kCaTop = 14;                        // exponent of the largest feature in an image, and of a row's largest query
constexpr int kCaSpread = 12;                     // rows of a tile whose exponents differ by more keep their own
constexpr int kCaSoftmax = 19;                    // pieces of a tile's softmax
constexpr int kCaLift = 11;                       // exponent that probabilities are lifted by: 2^(kCaMargin + kCaLift) fits fp16
static_assert(kCaLoads * 1024 * kCaWaves == kCaImage, "whole loads");
static_assert(kCaSlots * kCaImage <= 160 * 1024, "LDS of a CU");

// Place of piece j (8 features) of a tile's row t in its image, in 16-byte units. A key read takes one piece of 32
// consecutive rows; a value read takes four pieces of 4 rows at a time, which the XOR spreads over all banks.
KVIP_DEVICE int ca_place(int piece, int t) { return piece * kCaTile + (t ^ ((piece & 3) << 2)); }

// What the expanding launch leaves for the others.
struct ChunkPlan {
    int units;                                // workgroups with work
    int cut;                                  // tiles of a segment
    int cut_tiles;                            // row tiles, where they are cut; else 0
    int reserved;
    // In the order of the work, the longest contexts first:
    int units_before[KVIP_DRAFT_MAX_BATCH + 1];
    int tiles_before[KVIP_DRAFT_MAX_BATCH + 1];  // row tiles
    int4 request[KVIP_DRAFT_MAX_BATCH];          // first token, tokens, cached rows, first image (-1: none)
};

// Workspace: plan, then per image (rows with values that are no finite numbers, rows that are not there, code: four times
// the exponent, plus 2 where there are such rows, plus 1 where its rows have exponents of their own) and the rows'
// exponents, then the images, then the parts: 32 rows x 512 outputs of the part per wave as its lanes hold them
// ([block][quarter][lane] 16 bytes), then their (maximum, sum) pairs.
struct ChunkWork {
    ChunkPlan* plan;
    uint4* flags;
    int16_t* exponents;
    uint8_t* images;
    f32x4* outputs;
    float2* states;
};
__host__ __device__ inline int64_t ca_images(int64_t max_rows, int batch) { return (max_rows + kCaTile - 1) / kCaTile + batch; }
__host__ __device__ inline size_t ca_align(size_t n) { return (n + 1023) / 1024 * 1024; }
__host__ __device__ inline ChunkWork ca_work(void* base, int64_t images, size_t* bytes) {
    uint8_t* p = static_cast<uint8_t*>(base);
    size_t at = 0;
    auto take = [&](size_t n) {
        uint8_t* q = p + at;
        at = ca_align(at + n);
        return q;
    };
    ChunkWork w;
    w.plan = reinterpret_cast<ChunkPlan*>(take(sizeof(ChunkPlan)));
    w.flags = reinterpret_cast<uint4*>(take(static_cast<size_t>(images) * sizeof(uint4)));
    w.exponents = reinterpret_cast<int16_t*>(take(static_cast<size_t>(images) * kCaTile * sizeof(int16_t)));
    w.images = take(static_cast<size_t>(images) * kCaImage);
    w.outputs = reinterpret_cast<f32x4*>(take(static_cast<size_t>(kCaUnits) * kCaWaves * kCaBlocks * 4 * 64 * sizeof(f32x4)));
    w.states = reinterpret_cast<float2*>(take(static_cast<size_t>(kCaUnits) * kCaTileRows * sizeof(float2)));
    if (bytes != nullptr) *bytes = at;
    return w;
}

// A request as the kernels take it.
struct ChunkRequest {
    int begin;   // first token
    int tokens;
    int length;  // cached rows
    KVIP_DEVICE int past() const { return length - tokens; }
};
KVIP_DEVICE ChunkRequest ca_request(const KvipChunkAttnArgs& p, int b, uint32_t* err) {
    ChunkRequest q;
    const int first = p.cu_seqlens[b], behind = p.cu_seqlens[b + 1], given = p.seq_lens[b];
    const bool refused = p.steps != nullptr && p.steps[b] <= 0;
    q.begin = min(max(first, 0), p.max_tokens);
    q.tokens = min(max(behind, q.begin), p.max_tokens) - q.begin;
    q.length = refused ? 0 : min(max(given, 0), p.max_blocks * kBlockTokens);
    if (first != q.begin || behind != q.begin + q.tokens || (!refused && (given != q.length || (q.tokens > 0 && given < q.tokens)))) {
        *err |= KVIP_STATUS_BAD_LENGTH;
    }
    return q;
}
// Without the rows that an earlier request has, which come first (cu_seqlens that fall): `from` is the first row that is its own.
KVIP_DEVICE ChunkRequest ca_own(ChunkRequest q, int from) {
    const int taken = min(max(from - q.begin, 0), q.tokens);
    q.begin += taken;
    q.tokens -= taken;
    return q;
}
KVIP_DEVICE int ca_row_tiles(const ChunkRequest& q, int heads) { return (q.tokens * heads + kCaTileRows - 1) / kCaTileRows; }
KVIP_DEVICE int ca_steps(const ChunkRequest& q) { return q.tokens > 0 ? (q.length + kCaTile - 1) / kCaTile : 0; }

// Hardware round to nearest even.
KVIP_DEVICE uint32_t ca_pack(float a, float b) {
    const bf16x2 v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
    return __builtin_bit_cast(uint32_t, v);
}
KVIP_DEVICE uint32_t ca_pack_half(float a, float b) {
    const f16x2 v = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
    return __builtin_bit_cast(uint32_t, v);
}
// Exponent that takes the largest magnitude (of bits `most`, below infinity's) to 2^kCaTop .. 2^(kCaTop + 1); for images
// the next multiple of 4, so that most tiles have the same.
KVIP_DEVICE int ca_exponent(uint32_t most) { return static_cast<int>(most >> 23) - 127 - kCaTop; }
KVIP_DEVICE int ca_image_exponent(uint32_t most) { return (ca_exponent(most) + 3) & ~3; }

// Plan and images. Every workgroup sums the requests' tiles for itself; the first one leaves the plan, the others take
// images in turn. A thread takes 64 features of a row (16 of each scale group, so that 8 threads read whole lines) and 8
// rotary features.
__global__ __launch_bounds__(kCaThreads) void chunk_expand_kernel(const KvipChunkAttnArgs p) {
    __shared__ __align__(16) uint8_t s_image[kCaImage];
    __shared__ int s_before[KVIP_DRAFT_MAX_BATCH + 1];
    __shared__ uint32_t s_sums[kCaWaves];
    __shared__ uint4 s_flags[kCaWaves];
    constexpr int kPer = KVIP_DRAFT_MAX_BATCH / kCaThreads;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int64_t most = ca_images(p.max_rows, p.batch);
    const ChunkWork work = ca_work(p.workspace, most, nullptr);
    uint32_t err = 0;
    int steps[kPer];
    uint32_t sum = 0, sum_tiles = 0, total, total_tiles;
    bool fall = false;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int b = tid * kPer + i;
        steps[i] = 0;
        if (b < p.batch) {
            const ChunkRequest q = ca_request(p, b, &err);
            steps[i] = ca_steps(q);
            sum_tiles += ca_row_tiles(q, p.heads);
            fall |= p.cu_seqlens[b + 1] < p.cu_seqlens[b];
        }
        sum += steps[i];
    }
    uint32_t before = block_exclusive_scan(sum, s_sums, &total);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int b = tid * kPer + i;
        if (b <= p.batch) s_before[b] = before;
        before += steps[i];
    }
    if (tid == 0) s_before[p.batch] = total;
    __syncthreads();

    if (blockIdx.x == 0) {
        __shared__ int s_longest, s_steps[KVIP_DRAFT_MAX_BATCH], s_tiles[KVIP_DRAFT_MAX_BATCH + 1], s_units[kCaMostCuts];
        __shared__ unsigned long long s_work;  // tiles of all row tiles
        ChunkPlan* plan = work.plan;
        if (tid == 0) {
            s_longest = 1;
            s_work = 0;
        }
        if (tid < kCaMostCuts) s_units[tid] = 0;
        // Where cu_seqlens fall, several requests have the same rows, and the launches have no workgroups for more than max_tokens:
        // each row goes with the first of them. (The images are laid out all the same.)
        int* s_own = reinterpret_cast<int*>(s_image);  // first row of each request's own, where they fall
        const bool falls = __syncthreads_or(fall) != 0;
        if (falls) {
            if (tid == 0) {
                int behind = 0;
                for (int b = 0; b < p.batch; ++b) {
                    uint32_t none = 0;
                    const ChunkRequest q = ca_request(p, b, &none);
                    s_own[b] = behind;
                    behind = max(behind, q.begin + q.tokens);
                }
            }
            __syncthreads();
            sum_tiles = 0;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int b = tid * kPer + i;
                uint32_t none = 0;
                if (b < p.batch) sum_tiles += ca_row_tiles(ca_own(ca_request(p, b, &none), s_own[b]), p.heads);
            }
        }
        block_exclusive_scan(sum_tiles, s_sums, &total_tiles);
        // Requests by their context, the longest first, so that what is left at the end is short.
        for (int b = tid; b < p.batch; b += kCaThreads) {
            uint32_t none = 0;
            ChunkRequest q = ca_request(p, b, &none);
            const int steps_b = ca_steps(q);
            if (falls) q = ca_own(q, s_own[b]);
            int rank = 0;
            for (int i = 0; i < p.batch; ++i) {
                const int other = s_before[i + 1] - s_before[i];
                rank += other > steps_b || (other == steps_b && i < b);
            }
            // No images: none that would fit.
            const bool fits = s_before[b + 1] <= most;
            plan->request[rank] = make_int4(q.begin, q.tokens, q.length, fits ? s_before[b] : -1);
            if (!fits && steps_b > 0) err |= KVIP_STATUS_BAD_LENGTH;
            s_steps[rank] = steps_b;
            s_tiles[rank] = ca_row_tiles(q, p.heads);
            atomicMax(&s_longest, steps_b);
            // Half of the chunk's own rows is not seen.
            atomicAdd(&s_work, static_cast<unsigned long long>(s_tiles[rank]) * max(steps_b - q.tokens / (2 * kCaTile), 1));
        }
        __syncthreads();
        const int longest = s_longest;
        for (int b = tid / kCaMostCuts; b < p.batch && total_tiles <= kCaCutTiles; b += kCaThreads / kCaMostCuts) {
            const int k = tid % kCaMostCuts, c = (longest + k) / (k + 1);
            atomicAdd(&s_units[k], s_tiles[b] * max((s_steps[b] + c - 1) / c, 1));
        }
        __syncthreads();
        // The context is cut into k + 1 segments of the longest request's where that ends earlier: the workgroups come in
        // rounds of one per CU, or, where they are unequal, keep every CU busy but for half of one of them.
        int cut = longest;
        float best = 0.f;
        for (int k = 0; k < (total_tiles <= kCaCutTiles ? kCaMostCuts : 0); ++k) {
            const int c = (longest + k) / (k + 1), units = s_units[k];
            const float rounds = static_cast<float>((units + kCaCus - 1) / kCaCus * c), spread = static_cast<float>(s_work) / kCaCus + 0.5f * c;
            const float cost = fmaxf(fminf(rounds, spread), c) + (k > 0 ? kCaPartSteps * (1.f + static_cast<float>(units) / kCaCus) : 0.f);
            if (k == 0 || (units <= kCaUnits && cost < best)) {
                best = cost;
                cut = c;
            }
        }
        uint32_t mine = 0, mine_tiles = 0, total_units;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int r = tid * kPer + i;
            if (r >= p.batch) break;
            mine += s_tiles[r] * max((s_steps[r] + cut - 1) / cut, 1);
            mine_tiles += s_tiles[r];
        }
        uint32_t units_before = block_exclusive_scan(mine, s_sums, &total_units);
        uint32_t tiles_before = block_exclusive_scan(mine_tiles, s_sums, &total_tiles);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int r = tid * kPer + i;
            if (r >= p.batch) break;
            plan->units_before[r] = units_before;
            plan->tiles_before[r] = tiles_before;
            units_before += s_tiles[r] * max((s_steps[r] + cut - 1) / cut, 1);
            tiles_before += s_tiles[r];
        }
        if (tid == 0) {
            plan->units = total_units;
            plan->cut = cut;
            plan->cut_tiles = cut < longest ? total_tiles : 0;
            plan->units_before[p.batch] = total_units;
            plan->tiles_before[p.batch] = total_tiles;
        }
        report(p.status, err);
        return;
    }

    int b = 0;
    for (int image = blockIdx.x - 1; image < static_cast<int>(total) && image < most; image += gridDim.x - 1) {
        // The request: the last one whose images begin at or before this one (empty ones share its beginning).
        int lo = b, hi = p.batch - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (s_before[mid] <= image) lo = mid;
            else hi = mid - 1;
        }
        b = lo;
        if (s_before[b + 1] > most) continue;  // its request does not fit
        uint32_t none = 0;
        const ChunkRequest q = ca_request(p, b, &none);
        const int first = (image - s_before[b]) * kCaTile, t = tid >> 3, piece = tid & 7;
        const int page = p.block_table[static_cast<int64_t>(b) * p.max_blocks + first / kBlockTokens];
        const bool in_cache = static_cast<unsigned>(page) < static_cast<unsigned>(p.num_blocks);
        if (!in_cache && tid == 0) report(p.status, KVIP_STATUS_BAD_BLOCK);
        const bool there = in_cache && first + t < q.length;
        v4i raw[4] = {}, rope = {};
        f32x4 scale = {};
        if (there) {
            const uint8_t* row = p.kv_cache + page * p.kv_block_stride + static_cast<int64_t>(first % kBlockTokens + t) * p.row_stride;
#pragma unroll
            for (int k = 0; k < 4; ++k) raw[k] = *reinterpret_cast<const v4i*>(row + k * 128 + piece * 16);
            rope = *reinterpret_cast<const v4i*>(row + kCaValue + piece * 16);
            scale = *reinterpret_cast<const f32x4*>(row + kCaValue + 128);
        }
        float x[64];
        uint32_t most_bits = 0;
        bool odd = false;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int bytes = raw[i / 4][i % 4];
            x[4 * i] = __builtin_amdgcn_cvt_f32_fp8(bytes, 0) * scale[i / 4];
            x[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8(bytes, 1) * scale[i / 4];
            x[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8(bytes, 2) * scale[i / 4];
            x[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8(bytes, 3) * scale[i / 4];
        }
#pragma unroll
        for (int i = 0; i < 64; ++i) most_bits = max(most_bits, __float_as_uint(x[i]) & 0x7FFFFFFFu);
        odd = most_bits >= 0x7F800000u;
        // A row's 8 threads lie side by side: bit t of the flags of the whole tile.
        const uint64_t odd_lanes = __ballot(odd), gone_lanes = __ballot(!there);
        const bool zero = odd_lanes >> (lane & 56) & 0xFF;
        if (zero) most_bits = 0;
        float turned[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            turned[i] = bf16_to_float(static_cast<uint16_t>(static_cast<uint32_t>(rope[i / 2]) >> (16 * (i & 1))));
            const uint32_t bits = __float_as_uint(turned[i]) & 0x7FFFFFFFu;
            most_bits = max(most_bits, bits < 0x7F800000u ? bits : 0u);
        }
        const float most_row = group_max<8>(__uint_as_float(most_bits));  // of rows without a feature: 0
        const float most_wave = group_max<64>(most_row);
        const float least_wave = -group_max<64>(most_row > 0.f ? -most_row : -INFINITY);
        uint32_t odd_rows = 0, gone_rows = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            odd_rows |= ((odd_lanes >> (8 * i) & 0xFF) != 0 ? 1u : 0u) << i;
            gone_rows |= static_cast<uint32_t>(gone_lanes >> (8 * i) & 1) << i;
        }
        if (lane == 0) s_flags[w] = make_uint4(odd_rows, gone_rows, __float_as_uint(most_wave), __float_as_uint(least_wave));
        __syncthreads();  // and the image before is copied
        uint4 flags = make_uint4(0, 0, 0, 0x7F800000u);
#pragma unroll
        for (int i = 0; i < kCaWaves; ++i) {
            flags.x |= s_flags[i].x << (8 * i);
            flags.y |= s_flags[i].y << (8 * i);
            flags.z = max(flags.z, s_flags[i].z);
            flags.w = min(flags.w, s_flags[i].w);
        }
        // One exponent for all rows, unless that would cost the smaller ones their bits: what a token sees must not
        // depend on rows that it does not.
        const int tile_exponent = ca_image_exponent(flags.z);
        const bool spread = flags.z != 0 && tile_exponent - ca_image_exponent(flags.w) > kCaSpread;
        const int exponent = !spread ? tile_exponent : most_row > 0.f ? ca_image_exponent(__float_as_uint(most_row)) : -200;
        if (spread && piece == 0) work.exponents[static_cast<int64_t>(image) * kCaTile + t] = static_cast<int16_t>(exponent);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            v4i out;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                out[i] = static_cast<int>(ca_pack_half(ldexpf(x[8 * k + 2 * i], -exponent), ldexpf(x[8 * k + 2 * i + 1], -exponent)));
            }
            *reinterpret_cast<v4i*>(s_image + 16 * ca_place(k / 2 * 16 + piece * 2 + k % 2, t)) = zero ? v4i{0, 0, 0, 0} : out;
        }
        v4i out;
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = static_cast<int>(ca_pack_half(ldexpf(turned[2 * i], -exponent), ldexpf(turned[2 * i + 1], -exponent)));
        *reinterpret_cast<v4i*>(s_image + 16 * ca_place(kCaValue / 8 + piece, t)) = out;
        __syncthreads();
        v4i* to = reinterpret_cast<v4i*>(work.images + static_cast<int64_t>(image) * kCaImage);
#pragma unroll
        for (int i = 0; i < kCaImage / 16 / kCaThreads; ++i) to[tid + i * kCaThreads] = *reinterpret_cast<const v4i*>(s_image + 16 * (tid + i * kCaThreads));
        if (tid == 0) work.flags[image] = make_uint4(flags.x, flags.y, static_cast<uint32_t>(tile_exponent * 4 + ((flags.x | flags.y) != 0 ? 2 : 0) + (spread ? 1 : 0)), 0);
    }
}

KVIP_DEVICE float ca_half_max(float x) {  // over lanes l and l ^ 32
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
KVIP_DEVICE float ca_half_sum(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
KVIP_DEVICE float ca_share(float l) { return l > 0.f || l != l ? 1.f / l : 0.f; }
KVIP_DEVICE float ca_lse(float m, float l) {  // maximum in log2 units, sum (0 where the row sees nothing)
    return l > 0.f || l != l ? (m + __builtin_amdgcn_logf(l)) * kCaLn2 : -INFINITY;
}
KVIP_DEVICE void ca_store(const KvipChunkAttnArgs& p, int64_t at, f32x4 v) {
    if (p.output_dtype == KVIP_DTYPE_FP32) {
        *reinterpret_cast<f32x4*>(static_cast<float*>(p.output) + at) = v;
    } else {
        *reinterpret_cast<bf16x4*>(static_cast<__bf16*>(p.output) + at) = __builtin_convertvector(v, bf16x4);
    }
}

// Direct-to-LDS load from a wave-uniform address and a lane's offset below 2^32 (see lds_async.h).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// OFFSET moves both sides.
template <int OFFSET>
KVIP_DEVICE void ca_dma16(const uint8_t* base, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:%3" : : "s"(lds), "v"(offset), "s"(base), "n"(OFFSET) : "memory", "m0");
}
#pragma clang diagnostic pop

// Keeps an accumulator in accumulation registers from here to the next hold.
KVIP_DEVICE void ca_hold(v16f& acc) { asm volatile("" : "+a"(acc)); }

// f(0), f(1), ... of compile-time indices.
template <typename F, int... I>
KVIP_DEVICE void for_all(F&& f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}

// What a workgroup has of the plan: unit `at` (row tiles and their segments) or, for the join, row tile `at`. All of it is
// loaded at once, by the thread that finds it.
struct ChunkUnit {
    ChunkRequest q;
    int image0;     // -1: the request has none
    int rt, seg;
    int unit0;      // of the row tile's segment 0
    int segs;
    int cut;
};
KVIP_DEVICE bool ca_unit(const ChunkPlan* plan, int batch, int at, bool of_join, int* s_found, ChunkUnit* u) {
    const int4 head = *reinterpret_cast<const int4*>(plan);
    for (int r = threadIdx.x; r < batch; r += blockDim.x) {
        const int units0 = plan->units_before[r], units1 = plan->units_before[r + 1];
        const int tiles0 = plan->tiles_before[r], tiles1 = plan->tiles_before[r + 1];
        const int4 request = plan->request[r];
        const int first = of_join ? tiles0 : units0, behind = of_join ? tiles1 : units1;
        if (first <= at && at < behind) {
            const int tiles = tiles1 - tiles0, segs = (units1 - units0) / tiles;
            const int tile = of_join ? tiles - 1 - (at - tiles0) : (at - units0) / segs;  // in the order of the units
            s_found[0] = request.x;
            s_found[1] = request.y;
            s_found[2] = request.z;
            s_found[3] = request.w;
            s_found[4] = tiles - 1 - tile;  // the tiles that see most first
            s_found[5] = (at - units0) % segs;
            s_found[6] = units0 + tile * segs;
            s_found[7] = segs;
        }
    }
    if (at >= (of_join ? head.z : head.x)) return false;
    __syncthreads();
    auto found = [&](int i) { return __builtin_amdgcn_readfirstlane(s_found[i]); };
    u->q.begin = found(0);
    u->q.tokens = found(1);
    u->q.length = found(2);
    u->image0 = found(3);
    u->rt = found(4);
    u->seg = found(5);
    u->unit0 = found(6);
    u->segs = found(7);
    u->cut = __builtin_amdgcn_readfirstlane(head.y);
    return true;
}

// Tiles that a row tile's rows see.
KVIP_DEVICE int ca_reach(const ChunkRequest& q, int rt, int heads) {
    const int last = min((rt + 1) * kCaTileRows, q.tokens * heads) - 1;
    const int end = min(max(q.past() + last / heads + 1, 0), q.length);
    return (end + kCaTile - 1) / kCaTile;
}

__global__ __launch_bounds__(kCaThreads, 1) void chunk_attention_kernel(const KvipChunkAttnArgs p) {
    __shared__ __align__(1024) uint8_t s_ring[kCaSlots * kCaImage];
    __shared__ int s_found[8];
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const ChunkWork work = ca_work(p.workspace, ca_images(p.max_rows, p.batch), nullptr);
    ChunkUnit unit;
    if (!ca_unit(work.plan, p.batch, blockIdx.x, false, s_found, &unit)) return;
    const ChunkRequest& q = unit.q;
    const int image0 = unit.image0, cut = unit.cut;
    const int rows = q.tokens * p.heads, first_row = unit.rt * kCaTileRows + w * kCaRows;
    const int reach = image0 < 0 ? 0 : ca_reach(q, unit.rt, p.heads);
    const int t0 = unit.seg * cut, t1 = min(t0 + cut, reach);
    const bool whole = reach <= cut;
    const int hn = lane & 31, hk = lane >> 5;
    const int row = first_row + hn, node = min(row, rows - 1) / p.heads;
    const int64_t out_first = static_cast<int64_t>(q.begin) * p.heads + first_row;
    if (t0 >= t1) {
        if (unit.seg != 0 || reach > 0) return;  // nothing of the row tile is here
        for (int i = tid; i < kCaTileRows * (kCaValue / 4); i += kCaThreads) {  // rows that see nothing
            const int r = unit.rt * kCaTileRows + i / (kCaValue / 4);
            if (r < rows) ca_store(p, (static_cast<int64_t>(q.begin) * p.heads + r) * kCaValue + i % (kCaValue / 4) * 4, f32x4{0.f, 0.f, 0.f, 0.f});
        }
        if (p.lse != nullptr && hk == 0 && row < rows) p.lse[out_first + hn] = -INFINITY;
        return;
    }
    const int sees = min(max(q.past() + node + 1, 0), q.length);  // cached rows that the lane's row sees
    // The first tile that some row of the wave does not see whole.
    const int t_mask = min(max(q.past() + min(first_row, rows - 1) / p.heads + 1, 0), q.length) / kCaTile;
    const uint32_t ring = lds_addr(s_ring);
    auto slot_of = [&](int t) { return ring + ((t - t0) & (kCaSlots - 1)) * kCaImage; };
    // The wave's share of tile t's image (past the last tile: the last one again), in kCaLoads loads.
    const uint8_t* from;
    uint32_t to;
    auto aim = [&](int t) {
        from = work.images + static_cast<int64_t>(image0 + min(t, t1 - 1)) * kCaImage + w * (kCaLoads * 1024);
        to = slot_of(t) + w * (kCaLoads * 1024);
    };
    auto fetch = [&](auto which) {
        constexpr int i = decltype(which)::value;
        ca_dma16<i % 4 * 1024>(from + i / 4 * 4096, lane * 16, to + i / 4 * 4096);
    };
    // Queries of the wave's rows (rows past the last: the last again; their outputs are not written) come through a slot of its
    // own, in groups of 8 pieces x 32 rows, in which piece j of row r stands in place j ^ (r & 7) of the row's 8: whole lines
    // from memory, and reads of a piece of 32 rows on all banks. (130 tokens x 16 heads on 130 / 1030 / 4130 rows 19.7 / 23.5 / 36.4 us with loads of each lane's own
    // row, 17.3 / 22.1 / 34.9 so; nothing where every CU is busy.) The largest feature is looked for while they arrive.
    constexpr int kGroups = kCaPieces / 8, kGroupLoads = kCaRows / 8, kGroupFrags = 4;
    const uint32_t mine = ring + w * kCaImage;
    {
        const int last = max(rows - 1 - first_row, 0);  // row of the wave
        const uint8_t* query = reinterpret_cast<const uint8_t*>(p.query) + (static_cast<int64_t>(q.begin) * p.heads + min(first_row, rows - 1)) * (2 * kCaKey);
        uint32_t from_row[kGroupLoads];
#pragma unroll
        for (int k = 0; k < kGroupLoads; ++k) from_row[k] = min(8 * k + (lane >> 3), last) * (2 * kCaKey) + ((lane & 7) ^ (lane >> 3)) * 16;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
#pragma unroll
            for (int k = 0; k < kGroupLoads; ++k) ca_dma16<0>(query + g * 128, from_row[k], mine + (g * kGroupLoads + k) * 1024);
        }
    }
    v16f o[kCaBlocks];
#pragma unroll
    for (int f = 0; f < kCaBlocks; ++f) {
#pragma unroll
        for (int i = 0; i < 16; ++i) o[f][i] = 0.f;
        ca_hold(o[f]);
    }
    v4i qf[kCaFrags];  // fragment i: features 16 i + 8 (lane / 32) .. + 7
    u16x2 most_q = {};
    uint32_t piece_at[kGroupFrags];
#pragma unroll
    for (int i = 0; i < kGroupFrags; ++i) {
        piece_at[i] = mine + hn * 128 + ((2 * i + hk) ^ (hn & 7)) * 16;
        asm volatile("" : "+v"(piece_at[i]));
    }
    for_all([&](auto which) {
        constexpr int g = decltype(which)::value;
        asm volatile("s_waitcnt vmcnt(%0)" : : "n"((kGroups - 1 - g) * kGroupLoads) : "memory");
#pragma unroll
        for (int i = g * kGroupFrags; i < (g + 1) * kGroupFrags; ++i) {
            qf[i] = *(LdsV4i)(piece_at[i % kGroupFrags] + g * 4096);
#pragma unroll
            for (int j = 0; j < 4; ++j) most_q = __builtin_elementwise_max(most_q, __builtin_bit_cast(u16x2, qf[i][j] & 0x7FFF7FFF));
        }
        __builtin_amdgcn_sched_barrier(0);
    }, std::make_integer_sequence<int, kGroups>{});
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
#pragma unroll
    for (int t = 0; t < kCaSlots - 2; ++t) {
        aim(t0 + t);
        for_all(fetch, std::make_integer_sequence<int, kCaLoads>{});
    }
    // They become fp16 under an exponent of their row's, exactly but for features below 2^-28 of its largest. A negative
    // scale turns their signs.
    uint32_t most_bits = static_cast<uint32_t>(max(most_q[0], most_q[1])) << 16;
    most_bits = __float_as_uint(ca_half_max(__uint_as_float(most_bits < 0x7F800000u ? most_bits : 0u)));
    const int q_exponent = max(ca_exponent(most_bits), -126);
    const float q_factor = __uint_as_float(static_cast<uint32_t>(127 - q_exponent) << 23 | (p.scale < 0.f ? 0x80000000u : 0u));
#pragma unroll
    for (int i = 0; i < kCaFrags; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t pair = static_cast<uint32_t>(qf[i][j]);
            qf[i][j] = static_cast<int>(ca_pack_half(__uint_as_float(pair << 16) * q_factor, __uint_as_float(pair & 0xFFFF0000u) * q_factor));
        }
        asm volatile("" : "+v"(qf[i]));  // worked out here, not in the tile loop
    }
    int scale_exponent;  // the scale in log2 units is scale2 times 2 to this
    const float scale2 = frexpf(fabsf(p.scale), &scale_exponent) * kCaLog2e;
    float m_run = -INFINITY, l_sum = 0.f;
    v16f s;
    v4i pb[2];  // probabilities of the tile whose values come next

    // The codes of 64 tiles, which the lanes hold.
    int held_first = t0;
    int held = static_cast<int>(work.flags[image0 + min(t0 + lane, reach - 1)].z);
    asm volatile("" : "+v"(held));

    // Operands are read from LDS kAhead products before their use, across the borders of logits and values too.
    constexpr int kAhead = 4;
    v4i ring_of[kAhead];
    const uint32_t key_at[2] = {static_cast<uint32_t>(16 * ca_place(hk, hn)), static_cast<uint32_t>(16 * (ca_place(2 + hk, hn) - 2 * kCaTile))};
    const int vp = (lane >> 4 & 1) * 2 + (lane >> 1 & 1), vt = 4 * hk + (lane >> 2 & 3);  // piece of a block, row of eight
    const uint32_t value_at[2] = {static_cast<uint32_t>(16 * ca_place(vp, vt) + 8 * (lane & 1)),
                                  static_cast<uint32_t>(16 * ca_place(vp, vt + 8) + 8 * (lane & 1))};
    // Addresses of a tile's keys or values; opaque, so that the reads take their places as offsets.
    struct Base {
        uint32_t at[2];
    };
    auto base_of = [&](int t, const uint32_t (&at)[2]) {
        Base base = {{slot_of(t) + at[0], slot_of(t) + at[1]}};
        asm volatile("" : "+v"(base.at[0]), "+v"(base.at[1]));
        return base;
    };
    auto key = [&](const Base& base, int i) { ring_of[i % kAhead] = *(LdsV4i)(base.at[i & 1] + i * 1024); };
    auto value = [&](const Base& base, int i) {  // of product i: block i / 2, cached rows 16 (i % 2) .. + 15
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS16x4)(base.at[0] + (i >> 1) * 2048 + (i & 1) * 256));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS16x4)(base.at[1] + (i >> 1) * 2048 + (i & 1) * 256));
        ring_of[i % kAhead] = __builtin_bit_cast(v4i, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    static_assert(kCaFrags % kAhead == 0 && 2 * kCaBlocks % kAhead == 0, "the operand ring goes on at its start");
    // What the tile's flags and its place say. Features of a tile stand under its exponent, a row's sums under the largest
    // of the exponents that it has seen: a tile's probabilities take the difference, their sum gives it back.
    int exponent = -300, shift, lower;  // of the sums; by how much it has just risen; what the tile's is below it
    float factor;                       // from logits as they come to those in log2 units
    bool spread;                        // the tile's rows have exponents of their own
    auto row_exponent = [&](int t, int i) {
        return static_cast<int>(work.exponents[static_cast<int64_t>(image0 + t) * kCaTile + 8 * (i >> 2) + 4 * hk + (i & 3)]);
    };
    int of_tile, tile_exponent, calm = 0x7FFFFFFF;  // calm: the exponent that leaves these as they are
    bool special;
    auto look = [&](int t) {  // does not need the logits
        if (t >= held_first + 64) {
            held_first = t;
            held = static_cast<int>(work.flags[image0 + min(t + lane, reach - 1)].z);
            asm volatile("" : "+v"(held));  // waited for here, not at every use
        }
        const int code = __builtin_amdgcn_readlane(held, t - held_first);
        tile_exponent = code >> 2;
        spread = (code & 1) != 0;
        special = (code & 3) != 0 || t >= t_mask;
    };
    // Logits of a tile, whose first operands are under way; the loads that are aimed at stand between the products, the
    // first value operands of the tile at `next` behind them.
    auto logits = [&](int t, const Base& base, const Base& next) {
        for_all([&](auto which) {
            constexpr int i = decltype(which)::value;
            if constexpr (i == 0) {
                const v16f zero = {};
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, ring_of[i % kAhead]), __builtin_bit_cast(f16x8, qf[i]), zero, 0, 0, 0);
            } else {
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, ring_of[i % kAhead]), __builtin_bit_cast(f16x8, qf[i]), s, 0, 0, 0);
            }
            if constexpr (i + kAhead < kCaFrags) key(base, i + kAhead);
            else value(next, i + kAhead - kCaFrags);
            if constexpr (i % 4 == 0) fetch(std::integral_constant<int, i / 4>{});
            if constexpr (i == kCaFrags / 2) look(t);
            __builtin_amdgcn_sched_barrier(0);
        }, std::make_integer_sequence<int, kCaFrags>{});
    };
    static_assert(kCaLoads * 4 == kCaFrags, "a load every four products");
    auto mask = [&](int t) {
        of_tile = tile_exponent;
        if (special) {
            const uint4 flags = work.flags[image0 + t];
            const int left = sees - t * kCaTile;
            uint32_t seen = left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1;
            seen &= ~flags.y;
            if (seen & flags.x) l_sum = NAN;
            if (seen == 0) of_tile = exponent;
            seen >>= 4 * hk;
            if (spread) {
                int top = -300;
                for (int i = 0; i < 16; ++i) {
                    if (seen >> (8 * (i >> 2) + (i & 3)) & 1) top = max(top, row_exponent(t, i));
                }
                top = static_cast<int>(ca_half_max(static_cast<float>(top)));
                of_tile = top;
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = ldexpf(s[i], min(row_exponent(t, i) - top, 0));
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (!(seen >> (8 * (i >> 2) + (i & 3)) & 1)) s[i] = -INFINITY;
            }
        }
    };
    // Softmax of the logits, p = 2^(factor logit - m + kCaLift + lower), in kCaSoftmax pieces. Its factor for what came before
    // (alpha) counts once the values of the tile before are in.
    float mx, bias, alpha, fresh_sum;
    bool raise;
    auto softmax = [&](int piece) {
        if (piece == 0) {
            if (special || tile_exponent != calm) {
                shift = max(of_tile - exponent, 0);
                exponent += shift;
                lower = max(of_tile - exponent, -100);
                // A scale so small that the logits vanish still leaves a number, which what is masked stays below, and one so
                // large that they overflow leaves those that are 0.
                factor = fminf(fmaxf(ldexpf(scale2, scale_exponent + q_exponent + of_tile), 0x1p-126f), kCaLargest);
                calm = !spread && __ballot(shift != 0 || lower != 0 || of_tile != tile_exponent) == 0ull ? tile_exponent : 0x7FFFFFFF;
            }
        } else if (piece == 1) {
            mx = s[0];
#pragma unroll
            for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
            mx = ca_half_max(mx) * factor;
            fresh_sum = 0.f;
        } else if (piece == 2) {
            raise = mx - m_run > kCaMargin;  // also the first finite maximum
            const float m_new = raise ? mx : m_run;
            alpha = raise && m_run != -INFINITY ? __builtin_amdgcn_exp2f(m_run - m_new) : raise ? 0.f : 1.f;
            m_run = m_new;
            const float lift = static_cast<float>(kCaLift + lower);
            bias = (m_new == -INFINITY ? 0.f : -m_new) + lift;
            if (__ballot(fabsf(m_new) > 0x1p20f && m_new != -INFINITY) != 0ull) {
                // Logits whose rounding a fused product would show: the difference from the maximum, rounded as that was.
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float x = s[i] * factor;
                    asm volatile("" : "+v"(x));
                    s[i] = m_new == -INFINITY ? x : x - m_new;
                }
                factor = 1.f;
                bias = lift;
                calm = 0x7FFFFFFF;
            }
            asm volatile("" : "+v"(bias), "+v"(factor));
        } else {
            float p1 = __builtin_amdgcn_exp2f(fmaf(s[piece - 3], factor, bias));
            fresh_sum += p1;
            asm volatile("" : "+v"(p1), "+v"(fresh_sum));  // here, not behind the products
            s[piece - 3] = p1;
        }
    };
    auto take = [&](int t) {  // the softmax's results become those of tile t, whose values come next
        l_sum = l_sum * alpha + ldexpf(fresh_sum, -lower);
        if (spread) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = ldexpf(s[i], min(row_exponent(t, i) - (exponent + lower), 0));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) pb[i >> 2][i & 3] = static_cast<int>(ca_pack_half(s[2 * i], s[2 * i + 1]));
    };
    // Every load of the tile after next has landed but the last kCaLoads of this wave, and all reads of this wave are done;
    // then those of all waves.
    auto arrive = [&] {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"((kCaSlots - 3) * kCaLoads) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" : : : "memory");
    };
    // Values of a tile, whose first operands are under way, with the softmax of the next one beside them and the first key
    // operands of the one after that (at `next`) behind them: when the last reads are done, so is the tile.
    auto values = [&](const Base& base, const Base& next, auto with_softmax) {
        constexpr bool kSoftmax = decltype(with_softmax)::value;
        for_all([&](auto which) {
            constexpr int i = decltype(which)::value;
            if constexpr (i % 2 == 0) ca_hold(o[i / 2]);
            o[i / 2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, ring_of[i % kAhead]), __builtin_bit_cast(f16x8, pb[i % 2]), o[i / 2], 0, 0, 0);
            if constexpr (i % 2 == 1) ca_hold(o[i / 2]);
            if constexpr (i + kAhead < 2 * kCaBlocks) value(base, i + kAhead);
            else if constexpr (kSoftmax) {
                if constexpr (i + kAhead == 2 * kCaBlocks) arrive();
                key(next, i + kAhead - 2 * kCaBlocks);
            }
            if constexpr (kSoftmax) {  // over all products, once the logits are there
                constexpr int from = i * kCaSoftmax / (2 * kCaBlocks), to = (i + 1) * kCaSoftmax / (2 * kCaBlocks);
                if constexpr (to > from) softmax(from);
            }
            __builtin_amdgcn_sched_barrier(0);
        }, std::make_integer_sequence<int, 2 * kCaBlocks>{});
    };
    arrive();
    Base values_base = base_of(t0, value_at), keys_base = base_of(t0, key_at);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) key(keys_base, i);
    aim(t0 + kCaSlots - 2);
    logits(t0, keys_base, values_base);
    mask(t0);
#pragma unroll
    for (int i = 0; i < kCaSoftmax; ++i) softmax(i);
    take(t0);
    if (t0 + 1 < t1) {
        arrive();
        keys_base = base_of(t0 + 1, key_at);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) key(keys_base, i);
    }
#pragma unroll 1
    for (int t = t0; t + 1 < t1; ++t) {
        aim(t + kCaSlots - 1);
        const Base here = base_of(t, value_at), keys_next = base_of(t + 2, key_at);
        logits(t + 1, keys_base, here);
        mask(t + 1);
        values(here, keys_next, std::true_type{});
        keys_base = keys_next;
        if (__ballot(raise || shift != 0) != 0ull) {
            const float to_new = ldexpf(alpha, -shift);
#pragma unroll
            for (int f = 0; f < kCaBlocks; ++f) {
                ca_hold(o[f]);
                o[f] *= to_new;
                ca_hold(o[f]);
            }
        }
        take(t + 1);
    }
    values_base = base_of(t1 - 1, value_at);
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
#pragma unroll
    for (int i = 0; i < kAhead; ++i) value(values_base, i);
    values(values_base, values_base, std::false_type{});
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // the loads past the last tile

    const float l_all = ldexpf(ca_half_sum(l_sum), -kCaLift);
    // The smallest exponents are taken in two steps, so that the share is an ordinary number.
    const int below = min(exponent + 64, 0);
    if (__ballot(below != 0) != 0ull) {
#pragma unroll
        for (int f = 0; f < kCaBlocks; ++f) {
            ca_hold(o[f]);
            o[f] *= ldexpf(1.f, below);
            ca_hold(o[f]);
        }
    }
    const float share = ldexpf(ca_share(l_all), exponent - below - kCaLift);
    int hn_ = hn;
    asm volatile("" : "+v"(hn_));  // what comes of it is not held over the tile loop
    f32x4* part = work.outputs + (static_cast<int64_t>(blockIdx.x) * kCaWaves + w) * (kCaBlocks * 4 * 64) + lane;
#pragma unroll
    for (int f = 0; f < kCaBlocks; ++f) {
        ca_hold(o[f]);
        const v16f x = o[f] * share;
        if (!whole) {
#pragma unroll
            for (int a = 0; a < 4; ++a) part[(f * 4 + a) * 64] = f32x4{x[4 * a], x[4 * a + 1], x[4 * a + 2], x[4 * a + 3]};
        } else if (p.output_dtype == KVIP_DTYPE_BF16) {
            // The halves of the wave hold every other four features of a row: swapped, each has eight.
#pragma unroll
            for (int a = 0; a < 4; a += 2) {
                v4i v;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const auto pair = __builtin_amdgcn_permlane32_swap(
                        ca_pack(x[4 * a + 2 * e], x[4 * a + 2 * e + 1]), ca_pack(x[4 * a + 2 * e + 4], x[4 * a + 2 * e + 5]), false, false);
                    v[e] = pair[0];
                    v[e + 2] = pair[1];
                }
                if (hn_ < rows - first_row) *reinterpret_cast<v4i*>(static_cast<__bf16*>(p.output) + (out_first + hn_) * kCaValue + 32 * f + 8 * a + 8 * hk) = v;
            }
        } else if (hn_ < rows - first_row) {
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                ca_store(p, (out_first + hn_) * kCaValue + 32 * f + 8 * a + 4 * hk, f32x4{x[4 * a], x[4 * a + 1], x[4 * a + 2], x[4 * a + 3]});
            }
        }
    }
    if (hk == 0) {
        if (!whole) work.states[static_cast<int64_t>(blockIdx.x) * kCaTileRows + w * kCaRows + hn_] = make_float2(m_run, l_all);
        else if (p.lse != nullptr && hn_ < rows - first_row) p.lse[out_first + hn_] = ca_lse(m_run, l_all);
    }
}

// Joins the parts of row tiles that were cut. A workgroup takes one wave's 32 rows and a quarter of the features.
__global__ __launch_bounds__(kCaThreads) void chunk_join_kernel(const KvipChunkAttnArgs p) {
    __shared__ int s_found[8];
    const ChunkWork work = ca_work(p.workspace, ca_images(p.max_rows, p.batch), nullptr);
    const int slice = blockIdx.x % 4, rg = blockIdx.x / 4 % kCaWaves;
    ChunkUnit u;
    if (!ca_unit(work.plan, p.batch, blockIdx.x / 4 / kCaWaves, true, s_found, &u)) return;
    const ChunkRequest& q = u.q;
    const int rt = u.rt, unit = u.unit0, cut = u.cut;
    const int reach = u.image0 < 0 ? 0 : ca_reach(q, rt, p.heads);
    if (reach <= cut) return;  // whole
    const int parts = min((reach + cut - 1) / cut, u.segs);
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, hn = lane & 31;
    const int row = rt * kCaTileRows + rg * kCaRows + hn, rows = q.tokens * p.heads;
    const float2* states = work.states + static_cast<int64_t>(unit) * kCaTileRows + rg * kCaRows + hn;
    constexpr int kRun = kCaBlocks / 4;  // fours of features of a wave
    constexpr int kAtOnce = 4;           // parts whose loads are issued together
    const int at = (slice * kCaWaves + w) * kRun;
    const f32x4* outputs = work.outputs + (static_cast<int64_t>(unit) * kCaWaves + rg) * (kCaBlocks * 4 * 64) + at * 64 + lane;
    float m = -INFINITY, l = 0.f;
    f32x4 x[kRun] = {};
    for (int first = 0; first < parts; first += kAtOnce) {
        float2 state[kAtOnce];
        f32x4 y[kAtOnce][kRun];
        float most = m;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            state[i] = make_float2(-INFINITY, 0.f);
            if (first + i >= parts) continue;
            state[i] = states[(first + i) * kCaTileRows];
#pragma unroll
            for (int j = 0; j < kRun; ++j) y[i][j] = __builtin_nontemporal_load(outputs + (static_cast<int64_t>(first + i) * kCaWaves * (kCaBlocks * 4) + j) * 64);
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) most = fmaxf(most, state[i].x);
        const float keep = most == -INFINITY ? l : l * __builtin_amdgcn_exp2f(m - most);
        l = keep;
        float weight[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            // A part without a maximum has no outputs, but may be NaN as a whole.
            weight[i] = state[i].x == -INFINITY ? state[i].y : state[i].y * __builtin_amdgcn_exp2f(state[i].x - most);
            l += weight[i];
        }
        // Outputs so far are outputs, not sums: no row is too large for them.
        const float share = ca_share(l);
#pragma unroll
        for (int j = 0; j < kRun; ++j) x[j] *= keep * share;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            if (first + i >= parts) break;
#pragma unroll
            for (int j = 0; j < kRun; ++j) x[j] += y[i][j] * (weight[i] * share);
        }
        m = most;
    }
    const int64_t out_row = static_cast<int64_t>(q.begin) * p.heads + row;
    if (row >= rows) return;
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
        ca_store(p, out_row * kCaValue + (at + j) / 4 * 32 + (at + j) % 4 * 8 + (lane >> 5) * 4, x[j]);
    }
    if (slice == 0 && threadIdx.x < kCaRows && p.lse != nullptr) p.lse[out_row] = ca_lse(m, l);
}

int64_t ca_row_tiles_most(int batch, int heads, int max_tokens) {
    return (static_cast<int64_t>(max_tokens) * heads + kCaTileRows - 1) / kCaTileRows + batch;
}

bool ca_sizes(int32_t batch, int32_t heads, int32_t max_tokens, int64_t max_rows) {
    return batch >= 1 && batch <= KVIP_DRAFT_MAX_BATCH && heads >= 1 && heads <= 128 && max_tokens >= 1 &&
           max_tokens <= KVIP_DRAFT_MAX_TOKENS && max_rows >= 1 && max_rows <= (1ll << 31);
}

// Few rows of the problem per request are the business of kvip_hip_tree_attention, which reads the cache as it is: here
// the images cost 1808 bytes of traffic per cached row. One request of 16 heads on 16000 rows, 1 / 16 / 64 tokens: 25.6 / 46.9 /
// 69.7 us there, 52.3 / 55.1 / 69.8 here; of 128 heads, 4 / 16 / 64 tokens: 50.3 / 105 / 318 and 56.5 / 95.9 / 258; 8
// requests of 16 heads x 8 tokens on 8000 rows: 55.0 and 80.4, of 128 heads: 190 and 166. (A workspace of this file's, of 269 MB or
// more, would do there too: 135 MB at most. So a call may have a narrower block table than its workspace was sized for.)
bool ca_few(int32_t batch, int32_t heads, int32_t max_tokens, int32_t max_blocks) {
    return max_tokens <= KVIP_DRAFT_MAX_NODES && static_cast<int64_t>(max_tokens) * heads <= 512ll * batch &&
           kvip_hip_tree_attention_workspace_bytes(batch, heads, max_tokens, max_blocks) != 0;
}

}  // namespace
}  // namespace kvip

extern "C" uint64_t kvip_hip_chunk_attention_workspace_bytes(int32_t batch, int32_t heads, int32_t max_tokens, int32_t max_blocks,
                                                             int64_t max_rows) {
    if (!kvip::ca_sizes(batch, heads, max_tokens, max_rows) || max_blocks < 1 || max_blocks > (1 << 17)) return 0;
    if (kvip::ca_few(batch, heads, max_tokens, max_blocks)) {
        return kvip_hip_tree_attention_workspace_bytes(batch, heads, max_tokens, max_blocks);
    }
    size_t bytes;
    kvip::ca_work(nullptr, kvip::ca_images(max_rows, batch), &bytes);
    return bytes;
}

extern "C" uint32_t kvip_hip_chunk_attention(const KvipChunkAttnArgs* a, void* stream) {
    if (a == nullptr) return KVIP_ERR_INVALID;
    auto aligned = [](const void* x, unsigned n) { return (reinterpret_cast<uintptr_t>(x) & (n - 1)) == 0; };
    const bool ok = a->query && a->kv_cache && a->block_table && a->seq_lens && a->cu_seqlens && a->output && a->workspace &&
                    aligned(a->query, 16) && aligned(a->kv_cache, 16) && aligned(a->output, 16) && aligned(a->workspace, 16) &&
                    kvip::ca_sizes(a->batch, a->heads, a->max_tokens, a->max_rows) && a->max_blocks >= 1 &&
                    a->max_blocks <= (1 << 17) && a->num_blocks >= 1 && a->num_blocks < (1 << 24) &&
                    a->row_stride >= KVIP_KV_ROW_BYTES && a->row_stride <= (1 << 24) && a->row_stride % 16 == 0 &&
                    a->kv_block_stride % 16 == 0 && a->kv_block_stride >= static_cast<int64_t>(kvip::kBlockTokens) * a->row_stride &&
                    (a->output_dtype == KVIP_DTYPE_BF16 || a->output_dtype == KVIP_DTYPE_FP32) && a->scale - a->scale == 0.f;
    if (!ok) return KVIP_ERR_INVALID;
    if (kvip::ca_few(a->batch, a->heads, a->max_tokens, a->max_blocks)) {
        KvipTreeAttnArgs t = {};
        t.query = a->query;
        t.kv_cache = a->kv_cache;
        t.block_table = a->block_table;
        t.seq_lens = a->seq_lens;
        t.cu_seqlens = a->cu_seqlens;
        t.steps = a->steps;
        t.output = a->output;
        t.lse = a->lse;
        t.workspace = a->workspace;
        t.status = a->status;
        t.kv_block_stride = a->kv_block_stride;
        t.row_stride = a->row_stride;
        t.batch = a->batch;
        t.heads = a->heads;
        t.max_nodes = a->max_tokens;
        t.max_tokens = a->max_tokens;
        t.max_blocks = a->max_blocks;
        t.num_blocks = a->num_blocks;
        t.output_dtype = a->output_dtype;
        t.scale = a->scale;
        return kvip_hip_tree_attention(&t, stream);
    }
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t images = kvip::ca_images(a->max_rows, a->batch), tiles = kvip::ca_row_tiles_most(a->batch, a->heads, a->max_tokens);
    const int64_t units = tiles < kvip::kCaUnits ? kvip::kCaUnits : tiles;
    hipLaunchKernelGGL(kvip::chunk_expand_kernel, dim3(static_cast<unsigned>(images < 1024 ? images : 1024) + 1), dim3(kvip::kCaThreads), 0, s, *a);
    hipLaunchKernelGGL(kvip::chunk_attention_kernel, dim3(static_cast<unsigned>(units)), dim3(kvip::kCaThreads), 0, s, *a);
    const int64_t joined = tiles < kvip::kCaCutTiles ? tiles : kvip::kCaCutTiles;
    hipLaunchKernelGGL(kvip::chunk_join_kernel, dim3(static_cast<unsigned>(joined * kvip::kCaWaves * 4)), dim3(kvip::kCaThreads), 0, s, *a);
    return static_cast<uint32_t>(hipGetLastError());
}
