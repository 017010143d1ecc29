// Rows of a table by token, scaled, and the table's gradient, on the caller's device tensors.
//
//   forward    out[t] = scale * table[token_t]
//   backward   dtable[v] = scale * sum over the tokens t = v of dy[t], every row of the table written once, zeros where no token asks for it
//
// A token outside the table has a row of zeros and no gradient.  Both are bound by memory.  Backward, the tokens are sorted (op_sort.cuh, a stable sort by up
// to ten bits at a time), so that a row's tokens lie together in ascending order.  A warp takes a few table rows: it finds the first one's tokens in the sorted list,
// reads on from there and adds the tokens' rows in registers.  Where that would be a long chain (more than `piece` tokens: a few tokens make up much of any text or board), the list's
// pieces of that many tokens are added up by blocks of their own in the same launch, the last of which adds up the pieces.  Sums are fp32 in an order that depends
// on the tokens alone, so results repeat bit for bit.
//
// Measured: forward 262144 x 512 bf16 of 73305 rows 51 us (6.1 TB/s); gradient of 73305 x 768 fp32 from 131072 tokens 135 us: the sort 27, the rows 105 (5.4 TB/s, 18 % of the warps an SM can hold: 48 KB
// of rows on their way per block).
#include "op_bulk.cuh"
#include "op_sort.cuh"

#include <atomic>
#include <utility>

namespace {

#define EMBED_THREADS 128
#define EMBED_WARPS 4
// table rows per warp at most; with 8 of them, 16 and 32: 1000000 x 1 fp32 from 5000 tokens 66, 49 and 42 us, 200000 x 128 fp32 from 20000 47, 43 and 43, 73305 x 32 fp32 from 131072 44, 46 and 48; above 2 KB 8 are better
// (73305 x 1024 fp32 from 65536 141 and 154)
#define EMBED_ROWS 16
#define EMBED_NAN __int_as_float(0x7fc00000)  // what sums are after a wait that has run out

struct Tokens {
    const void* p;
    int wide;  // 64-bit ones
    int64_t rows;
    // -1 where the table has no such row
    __device__ __forceinline__ int operator()(int64_t i) const {
        int64_t t;
        if (wide) t = static_cast<const int64_t*>(p)[i];
        else t = static_cast<const int*>(p)[i];
        return t >= 0 && t < rows ? (int)t : -1;
    }
};

// ---- forward ---------------------------------------------------------------------------------------------------------------
// L lanes take CH * VEC columns each of R tokens' rows
template <typename T, int VEC, int L, int CH, int R>
__global__ void __launch_bounds__(EMBED_THREADS)
k_embed_forward(Tokens tokens, int64_t count, const T* table, int64_t table_stride, int n, int tiles, float scale, T* __restrict__ out, int64_t out_stride) {
    const int64_t unit = (int64_t)blockIdx.x * (EMBED_THREADS / L) + threadIdx.x / L, group = unit / tiles;
    const int t = threadIdx.x % L, first = ((int)(unit - group * tiles) * (L * CH) + t) * VEC;
    op_next_may_start();
    op_wait_for_previous();
    int token[R];
#pragma unroll
    for (int q = 0; q < R; ++q) token[q] = group * R + q < count ? tokens(group * R + q) : -1;
    OpRaw<T, VEC> v[R][CH];
#pragma unroll
    for (int q = 0; q < R; ++q)
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = first + c * L * VEC;
            v[q][c].zero();
            if (token[q] >= 0 && col < n) v[q][c].load(table + token[q] * table_stride + col);
        }
#pragma unroll
    for (int q = 0; q < R; ++q)
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = first + c * L * VEC;
            float o[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) o[i] = token[q] >= 0 ? v[q][c].get(i) * scale : 0.0f;
            if (group * R + q < count && col < n) op_store<T, VEC>(out + (group * R + q) * out_stride + col, o);
        }
}

// ---- the sort ----------------------------------------------------------------------------------------------------------------
// the first digits, of the tokens themselves; a token outside the table is -1 and has no place
struct FirstSource {
    Tokens tokens;
    int mask;
    __device__ __forceinline__ int operator()(int64_t i) const { return tokens(i); }
    __device__ __forceinline__ int id(int64_t i) const { return (int)i; }
    __device__ __forceinline__ int key(int v) const { return v < 0 ? -1 : v & mask; }
};
// counts for the sort by the next digits while the entries are placed: the blocks of that sort take `piece` places each.  (A launch of its own for it: 6 us.)
struct NextCount {
    int* part;  // NULL: none
    int keys, piece, shift;
    __device__ __forceinline__ void operator()(int v, int place) const {
        if (part) atomicAdd(part + (int64_t)(place / piece) * keys + (v >> shift & (keys - 1)), 1);
    }
};
struct FirstPut {
    int *key, *id, *count;  // count: of the tokens in the table
    int* zero;              // set to zero by a single block; by the launch that counts where there are more
    int64_t zeros;
    NextCount next;
    __device__ __forceinline__ void operator()(int i, int v, int place) const {
        if (place < 0) return;
        key[place] = v;
        id[place] = i;
        next(v, place);
    }
    __device__ __forceinline__ void rest(const int*, const int* begin, const SortPlan& p) const {
        if (blockIdx.x == 0 && threadIdx.x == 0) *count = begin[p.keys];
        for (int64_t i = threadIdx.x; gridDim.x == 1 && i < zeros; i += SORT_THREADS) zero[i] = 0;
    }
};
// further digits, of what the digits before have sorted
struct NextSource {
    const int *sorted, *ids, *count;
    int shift, mask;
    __device__ __forceinline__ int operator()(int64_t i) const {
        const int v = sorted[i];  // behind the last one anything
        return i < *count ? v : -1;
    }
    __device__ __forceinline__ int id(int64_t i) const { return ids[i]; }
    __device__ __forceinline__ int key(int v) const { return v < 0 ? -1 : v >> shift & mask; }
};
struct NextPut {
    int *key, *id;
    NextCount next;
    __device__ __forceinline__ void operator()(int i, int v, int place) const {
        if (place < 0) return;
        key[place] = v;
        id[place] = i;
        next(v, place);
    }
    __device__ __forceinline__ void rest(const int*, const int*, const SortPlan&) const {}
};

// The first of the sorted keys [from, to) that is v or more (to: none), by a warp: 32 of them are looked at at once
__device__ __forceinline__ int embed_below(const int* key, int from, int to, int v, int lane) {
    unsigned lo = (unsigned)from, hi = (unsigned)to;
    while (lo < hi) {
        const unsigned step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step - 1;  // below 2^32
        const unsigned below = __popc(__ballot_sync(0xffffffffu, at < hi && key[at] < v));
        hi = min(hi, lo + (below + 1) * step - 1);
        lo += below * step;
    }
    return (int)lo;
}

template <typename O, int VEC>
__device__ __forceinline__ void embed_store(O* p, const float (&from)[VEC]) {
    constexpr int STEP = VEC * sizeof(O) > 16 ? 16 / (int)sizeof(O) : VEC;
#pragma unroll
    for (int i = 0; i < VEC; i += STEP) {
        float t[STEP];
#pragma unroll
        for (int k = 0; k < STEP; ++k) t[k] = from[i + k];
        op_store<O, STEP>(p + i, t);
    }
}

template <int VEC, int CH>
__device__ __forceinline__ void embed_zero(float (&acc)[CH][VEC]) {
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[c][i] = 0.0f;
}

struct EmbedList {
    const int *key, *id, *count;   // count: of the tokens in the table
    int piece, pieces, together;   // tokens to a piece, how many pieces there can be, and how many of them a block looks at
    float* part;                   // [pieces][2][n]: the chunks' sums, at the piece and the end of it (first or last token) where the list's entries in the chunk begin
    int* done;                     // [pieces][2][tiles]: how many of a list's sums are there, counted at its first one; zero at the start
};

// acc += sums that other blocks have written
template <int VEC>
__device__ __forceinline__ void embed_add_sums(float (&acc)[VEC], const float* from) {
    if constexpr (VEC == 1) {
        acc[0] += __ldcg(from);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(from + i));
            acc[i] += v.x, acc[i + 1] += v.y, acc[i + 2] += v.z, acc[i + 3] += v.w;
        }
    }
}

// How a warp gets the rows of a window of the list, `here` of them by the lanes' ids: f(j) for each in order, with its columns added to acc on the way.
//
// By asynchronous copies: several are on their way for every warp whatever the lists' lengths, without registers.  Of a row that starts anywhere (VEC = 1) the 16-byte
// pieces that hold its columns are copied, and its columns are read from where they lie in them.
template <typename T, int VEC, int CH, int K>
struct EmbedCopies {
    static constexpr int TILE = 32 * VEC * CH, SLOT = TILE * (int)sizeof(T) + (VEC == 1 ? 16 : 0), SMEM = EMBED_WARPS * K * SLOT;
    static_assert(K * sizeof(T) >= 4, "the warps' sums lie in the same memory");
    // blocks per SM: what registers and memory allow
    static constexpr int PER_SM = CH * VEC <= 8 && SMEM <= 24 * 1024 ? 8 : CH * VEC <= 16 ? 6 : 4;
    BulkRing<K, SLOT> ring;
    unsigned char* memory;
    const T* dy;
    int64_t stride;
    unsigned bytes;
    __device__ __forceinline__ EmbedCopies(unsigned char* smem, uint64_t* bars, const T* rows, int64_t row_stride, int column, int n)
        : ring(smem + (threadIdx.x >> 5) * K * SLOT, bars + (threadIdx.x >> 5) * K), memory(smem + (threadIdx.x >> 5) * K * SLOT), dy(rows + column), stride(row_stride),
          bytes((unsigned)(min(TILE, n - column) * (int)sizeof(T))) {}
    __device__ __forceinline__ unsigned off(const T* row) const { return VEC == 1 ? (unsigned)(uintptr_t)row & 15u : 0u; }
    template <typename F>
    __device__ __forceinline__ void add(float (&acc)[CH][VEC], int id, int here, F f) {
        const int lane = threadIdx.x & 31;
        int sent = 0;
        for (int j = 0; j < here; ++j) {
            for (; sent < here && sent < j + K; ++sent) {
                const T* row = dy + __shfl_sync(0xffffffffu, id, sent) * stride;
                ring.put(reinterpret_cast<const unsigned char*>(row) - off(row), VEC == 1 ? (bytes + off(row) + 15u) & ~15u : bytes);
            }
            f(j);
            const unsigned from = VEC == 1 ? off(dy + __shfl_sync(0xffffffffu, id, j) * stride) : 0u;
            const T* x = reinterpret_cast<const T*>(memory + ring.take() * SLOT + from) + lane * VEC;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                OpRaw<T, VEC> v;
                v.load(x + c * 32 * VEC);
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[c][i] += v.get(i);
            }
            __syncwarp();
        }
    }
    __device__ __forceinline__ bool failed() const { return !ring.ok; }  // a wait has run out: of all sums from here on
    __device__ __forceinline__ void end() { ring.end(); }
};
// Through registers, K rows at a time: less latency where a warp has a few rows, and as many short ones as there are (an SM starts a copy every 90 cycles or so).
template <typename T, int VEC, int CH, int K>
struct EmbedLoads {
    static constexpr int TILE = 32 * VEC * CH, SMEM = EMBED_WARPS * TILE * 4;
    static constexpr int HELD = K * CH * ((VEC * (int)sizeof(T) + 3) / 4) + CH * VEC;  // registers
    static constexpr int PER_SM = HELD <= 28 ? 8 : HELD <= 48 ? 6 : 4;
    const T* dy;
    int64_t stride;
    int n;  // columns from the tile's first
    __device__ __forceinline__ EmbedLoads(unsigned char*, uint64_t*, const T* rows, int64_t row_stride, int column, int columns) : dy(rows + column), stride(row_stride), n(columns - column) {}
    template <typename F>
    __device__ __forceinline__ void add(float (&acc)[CH][VEC], int id, int here, F f) {
        const int lane = threadIdx.x & 31;
        for (int j0 = 0; j0 < here; j0 += K) {
            OpRaw<T, VEC> x[K][CH];
#pragma unroll
            for (int u = 0; u < K; ++u) {
                const T* row = dy + __shfl_sync(0xffffffffu, id, j0 + u) * stride;
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const int col = (c * 32 + lane) * VEC;
                    x[u][c].zero();
                    if (j0 + u < here && col < n) x[u][c].load(row + col);
                }
            }
#pragma unroll
            for (int u = 0; u < K; ++u) {
                if (j0 + u >= here) break;
                f(j0 + u);
#pragma unroll
                for (int c = 0; c < CH; ++c)
#pragma unroll
                    for (int i = 0; i < VEC; ++i) acc[c][i] += x[u][c].get(i);
            }
        }
    }
    __device__ __forceinline__ bool failed() const { return false; }
    __device__ __forceinline__ void end() {}
};

// The first blocks: a chunk of `together` pieces of the list and a tile of columns.  The others: `per` table rows and a tile per warp; it looks for the first row's place in the
// list once and reads on from there, 32 entries at a time.
template <typename T, typename O, int VEC, int CH, int K, template <typename, int, int, int> class Rows>
__global__ void __launch_bounds__(EMBED_THREADS, Rows<T, VEC, CH, K>::PER_SM)
k_embed_rows(const T* dy, int64_t dy_stride, EmbedList list, int64_t rows, int n, int tiles, int per, float scale, O* __restrict__ out, int64_t out_stride) {
    constexpr int TILE = 32 * VEC * CH;
    extern __shared__ __align__(128) unsigned char s_rows[];
    __shared__ uint64_t s_bars[EMBED_WARPS * K];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, piece_blocks = (list.pieces + list.together - 1) / list.together * tiles;
    op_next_may_start();
    const bool piece_block = (int64_t)blockIdx.x < piece_blocks;
    const int64_t unit = piece_block ? (int64_t)blockIdx.x : ((int64_t)blockIdx.x - piece_blocks) * EMBED_WARPS + warp, group = unit / tiles;
    const int column = (int)(unit - group * tiles) * TILE, first = column + lane * VEC;
    Rows<T, VEC, CH, K> from_rows(s_rows, s_bars, dy, dy_stride, column, n);
    op_wait_for_previous();
    const int count = *list.count;
    float acc[CH][VEC];
    embed_zero(acc);
    if (!piece_block) {
        const int64_t row0 = group * per;
        if (row0 >= rows) return;
        const int end_row = (int)min(row0 + per, rows);
        const auto store = [&](int64_t v) {
            const float by = from_rows.failed() ? EMBED_NAN : scale;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int col = first + c * 32 * VEC;
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[c][i] *= by;
                if (col < n) embed_store<O, VEC>(out + v * out_stride + col, acc[c]);
            }
            embed_zero(acc);
        };
        int v = (int)row0, last = -1;  // acc is v's; the key before the window
        for (int at = embed_below(list.key, 0, count, v, lane);;) {
            const int key = lane < count - at ? list.key[at + lane] : INT32_MAX, id = lane < count - at ? list.id[at + lane] : 0;
            const int ahead = list.piece < count - at - lane ? list.key[at + list.piece + lane] : -1, before = __shfl_up_sync(0xffffffffu, key, 1);
            // up to the window's first list that is longer than a piece, which is added up by pieces
            const unsigned longer = __ballot_sync(0xffffffffu, ahead == key && key != (lane ? before : last) && key < end_row);
            const int mine = __popc(__ballot_sync(0xffffffffu, key < end_row)), here = longer ? __ffs(longer) - 1 : mine;
            from_rows.add(acc, id, here, [&](int j) {
                const int k = __shfl_sync(0xffffffffu, key, j);
                for (; v < k; ++v) store(v);
            });
            if (longer) {
                last = __shfl_sync(0xffffffffu, key, here);
                for (; v < last; ++v) store(v);
                ++v;
                at = embed_below(list.key, at + here, count, v, lane);
            } else {
                if (mine < 32) break;
                last = __shfl_sync(0xffffffffu, key, 31);
                at += 32;
            }
        }
        for (; v < end_row; ++v) store(v);
        from_rows.end();
        return;
    }
    // Every warp looks at a piece: its first and its last token, and whether their lists are longer than a piece.
    struct Sum {
        int token, from, to, first, last;  // the token's entries in this piece, the list's first sum, which is in the chunk where it begins, and its last piece
    };
    __shared__ Sum s_sums[EMBED_WARPS][2];
    __shared__ bool s_last, s_failed;
    const int piece = (int)group * list.together + warp;
    if (threadIdx.x == 0) s_failed = false;
    if (lane == 0) s_sums[warp][0].token = s_sums[warp][1].token = -1;
    if (warp < list.together && (int64_t)piece * list.piece < count) {
        const int from = piece * list.piece, to = list.piece < count - from ? from + list.piece : count, first_key = list.key[from], last_key = list.key[to - 1];
        for (int slot = 0; slot < (first_key == last_key ? 1 : 2); ++slot) {
            const int v = slot ? last_key : first_key;
            const int b = slot ? embed_below(list.key, from, to, v, lane) : from, e = slot || last_key == v ? to : embed_below(list.key, from, to, v + 1, lane);
            const bool begins = slot || from == 0 || list.key[from - 1] != v;
            const bool longer = begins ? list.piece < count - b && list.key[b + list.piece] == v : e - from == list.piece || list.key[e - 1 - list.piece] == v;
            if (!longer) continue;
            const int begin = begins ? b : embed_below(list.key, 0, from, v, lane), end = e < to ? e : embed_below(list.key, to, count, v + 1, lane);
            // a list that begins inside a piece is that piece's last one
            if (lane == 0) s_sums[warp][slot] = {v, b, e, begin / list.piece * 2 + (begin % list.piece ? 1 : 0), (end - 1) / list.piece};
        }
    }
    __syncthreads();
    float* s_part = reinterpret_cast<float*>(s_rows);  // what the rows have come through
    // The warps' sums of their columns, added up in order: column at of the tile.  After a wait that has run out in any warp, copies may still have been on their way to where the sums
    // lie; they are waited for, and what the block puts out from there on is NaN by a mark that lies elsewhere.
    const auto share_out = [&](auto put) {
        from_rows.end();
        if (from_rows.failed()) s_failed = true;
        __syncthreads();
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < VEC; ++i) s_part[warp * TILE + (c * VEC + i) * 32 + lane] = acc[c][i];
        __syncthreads();
        for (int at = threadIdx.x; at < TILE; at += EMBED_THREADS) {
            float sum = s_part[at];
#pragma unroll
            for (int w = 1; w < EMBED_WARPS; ++w) sum += s_part[w * TILE + at];
            const int col = column + (at / 32 / VEC * 32 + at % 32) * VEC + at / 32 % VEC;
            if (col < n) put(col, s_failed ? EMBED_NAN : sum);
        }
    };
    for (int which = 0, next; which < 2 * list.together; which = next) {
        Sum sum = s_sums[which / 2][which % 2];
        next = which + 1;
        if (sum.token < 0) continue;
        // the list's entries in the further pieces of this chunk follow
        for (; next < 2 * list.together; ++next) {
            const Sum more = s_sums[next / 2][next % 2];
            if (more.token >= 0 && more.token != sum.token) break;
            if (more.token >= 0) sum.to = more.to;
        }
        const int64_t number = 2 * (group * list.together + which / 2) + which % 2;
        const int share = (sum.to - sum.from + EMBED_WARPS - 1) / EMBED_WARPS, mine_to = min(sum.from + (warp + 1) * share, sum.to);
        embed_zero(acc);
        for (int i0 = sum.from + warp * share; i0 < mine_to; i0 += 32) {
            const int many = min(32, mine_to - i0), id = lane < many ? list.id[i0 + lane] : 0;
            from_rows.add(acc, id, many, [](int) {});
        }
        share_out([&](int col, float x) { list.part[number * n + col] = x; });
        // who writes the list's last sum adds them all up
        __threadfence();
        __syncthreads();
        const int chunk = sum.first / 2 / list.together, sums = sum.last / list.together - chunk + 1;
        if (threadIdx.x == 0) s_last = atomicAdd(list.done + (int64_t)sum.first * tiles + column / TILE, 1) == sums - 1;
        __syncthreads();
        if (s_last) {
            __threadfence();
            embed_zero(acc);
            const int mine = (sums + EMBED_WARPS - 1) / EMBED_WARPS, to = min((warp + 1) * mine, sums);
#pragma unroll 4
            for (int k = warp * mine; k < to; ++k) {
                const float* from = list.part + (int64_t)(k == 0 ? sum.first : (chunk + k) * list.together * 2) * n;
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const int col = first + c * 32 * VEC;
                    if (col < n) embed_add_sums<VEC>(acc[c], from + col);
                }
            }
            share_out([&](int col, float x) { out[(int64_t)sum.token * out_stride + col] = op_round<O>(x * scale); });
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // copies may follow
        __syncthreads();
    }
    from_rows.end();
}

// Few tokens and a small table: a block per table row and tile looks through all tokens for its own, in order, and its warps take a share of them each.  One launch and
// no workspace; 1000 tokens, 81 x 256 fp32: 3.7 us, by the sort 12 to 14.
#define EMBED_FEW 2048
#define EMBED_FEW_WARPS 8
template <typename T, typename O, int VEC>
__global__ void __launch_bounds__(EMBED_FEW_WARPS * 32)
k_embed_few(Tokens tokens, int count, const T* dy, int64_t dy_stride, int n, int tiles, float scale, O* __restrict__ out, int64_t out_stride) {
    constexpr int TILE = 32 * VEC, STEPS = 4;
    __shared__ float s_part[EMBED_FEW_WARPS * TILE];
    __shared__ int s_id[EMBED_FEW], s_many[EMBED_FEW_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.x / tiles, column = (int)(blockIdx.x - row * tiles) * TILE;
    op_next_may_start();
    op_wait_for_previous();
    // a warp's eighth of the tokens, STEPS * 32 of them at a time
    const int rounds = (count + EMBED_FEW_WARPS * STEPS * 32 - 1) / (EMBED_FEW_WARPS * STEPS * 32);
    unsigned found[STEPS];
    int many = 0, at = 0, all = 0;
    const auto look = [&](int round) {
        int token[STEPS];  // on their way together
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int i = ((warp * rounds + round) * STEPS + s) * 32 + lane;
            token[s] = tokens(min(i, count - 1));
            if (i >= count) token[s] = -1;
        }
#pragma unroll
        for (int s = 0; s < STEPS; ++s) found[s] = __ballot_sync(0xffffffffu, token[s] == row);
    };
    for (int round = 0; round < rounds; ++round) {
        look(round);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) many += __popc(found[s]);
    }
    if (lane == 0) s_many[warp] = many;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < EMBED_FEW_WARPS; ++w) {
        at += w < warp ? s_many[w] : 0;
        all += s_many[w];
    }
    for (int round = 0; round < rounds; ++round) {
        if (rounds > 1) look(round);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            if (found[s] >> lane & 1) s_id[at + __popc(found[s] & ((1u << lane) - 1u))] = ((warp * rounds + round) * STEPS + s) * 32 + lane;
            at += __popc(found[s]);
        }
    }
    __syncthreads();
    float acc[1][VEC];
    embed_zero(acc);
    EmbedLoads<T, VEC, 1, 8> from_rows(nullptr, nullptr, dy, dy_stride, column, n);
    const int share = (all + EMBED_FEW_WARPS - 1) / EMBED_FEW_WARPS, to = min((warp + 1) * share, all);
    for (int i0 = warp * share; i0 < to; i0 += 32) {
        const int here = min(32, to - i0), id = lane < here ? s_id[i0 + lane] : 0;
        from_rows.add(acc, id, here, [](int) {});
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) s_part[warp * TILE + lane * VEC + i] = acc[0][i];
    __syncthreads();
    for (int k = threadIdx.x; k < TILE; k += EMBED_FEW_WARPS * 32) {
        float sum = s_part[k];
#pragma unroll
        for (int w = 1; w < EMBED_FEW_WARPS; ++w) sum += s_part[w * TILE + k];
        if (column + k < n) out[(int64_t)row * out_stride + column + k] = op_round<O>(sum * scale);
    }
}

// ---- plans -------------------------------------------------------------------------------------------------------------------
struct EmbedPlan {
    bool few;            // no sort
    int passes, bits;    // of the sort
    SortPlan sort;
    int piece, pieces;
    int64_t tables, done, words, list; // 32-bit ones of the sorts' counts, of the counted sums, of both and the count; of each sorted list, behind which the pieces' sums lie
};
bool embed_plan(int64_t count, int64_t rows, int n, EmbedPlan* p) {
    if (count < 0 || count > OP_MAX_ENTRIES || rows < 1 || rows > INT32_MAX || n < 1 || n > OP_MAX_COLUMNS) return false;
    // Every row's blocks look through all tokens: as long as they, and what they read, are less than the sort's launches.  They are counted as tiles of 128 columns, which is what fp32 rows of whole 16-byte
    // accesses have, because the workspace's size may depend neither on the type nor on the alignment; 16-bit rows have half as many blocks, and rows that start anywhere four times as many (9 tokens,
    // 122 x 1473 bf16: 12 us).
    const int64_t blocks = rows * ceil_div64(n, 128);
    p->few = count > 0 && count <= EMBED_FEW && blocks <= 16 * (int64_t)sm_count() && blocks * count <= 16 * 1024 * (int64_t)sm_count();
    int bits = 1;
    while (((int64_t)1 << bits) < rows) ++bits;
    p->passes = (bits + 9) / 10;
    p->bits = (bits + p->passes - 1) / p->passes;
    p->sort = sort_plan(count, 1 << p->bits, 1);
    // pieces of 32 tokens, or more where there were over 4096 of them: their sums are one chain per warp when they are joined
    p->piece = 32;
    while (count > (int64_t)p->piece * 4096) p->piece *= 2;
    p->pieces = (int)((count + p->piece - 1) / p->piece);
    p->list = (count + 7) / 8 * 8;
    // what one launch takes; tensors that fit a GPU are far below
    const int64_t tiles = ceil_div64(n, 32);
    if ((p->pieces + rows / EMBED_WARPS + 2) * tiles > INT32_MAX) return false;
    // the tables of counts, those of the sums that are there, the count of tokens
    p->tables = p->passes * sort_words(p->sort);
    p->done = (int64_t)p->pieces * 2 * tiles;
    p->words = (p->tables + p->done + 1 + 7) / 8 * 8;
    return true;
}
int64_t embed_bytes(const EmbedPlan& p, int n) { return p.few ? 0 : 4 * (p.words + (p.passes > 1 ? 4 : 2) * p.list + (int64_t)p.pieces * 2 * n); }

struct EmbedBackward {
    cudaStream_t s;
    Tokens tokens;
    int64_t count;
    bool few;
    const void* dy;
    int64_t dys, rows;
    int n;
    float scale;
    void* out;
    int64_t os;
    EmbedList list;
};
template <typename T, typename O, int VEC, int CH, int K, template <typename, int, int, int> class Rows = EmbedCopies>
void embed_rows_go(const EmbedBackward& a) {
    constexpr int SMEM = Rows<T, VEC, CH, K>::SMEM, PER_SM = Rows<T, VEC, CH, K>::PER_SM;
    const int tiles = (int)ceil_div64(a.n, 32 * VEC * CH);
    const auto kernel = k_embed_rows<T, O, VEC, CH, K, Rows>;
    if (SMEM > 40 * 1024) {
        static std::atomic<uint64_t> known{0};
        op_allow_smem(kernel, SMEM, known);
    }
    // Several rows per warp share the search: as many as leave every warp four turns, or one turn of short rows, which take no longer than the search.
    const int64_t turns = a.rows * tiles / ((int64_t)sm_count() * PER_SM * EMBED_WARPS * (a.n <= 256 / (int)sizeof(T) ? 1 : 4));
    const int per = (int)(turns < 1 ? 1 : turns > EMBED_ROWS ? EMBED_ROWS : turns);
    // pieces together where they are more than a few blocks per SM: most of them have no long list, and a long one has fewer sums
    EmbedList list = a.list;
    const int64_t many = (int64_t)list.pieces * tiles / (2 * sm_count());
    list.together = (int)(many < 1 ? 1 : many > EMBED_WARPS ? EMBED_WARPS : many);
    const int64_t blocks = ceil_div64(list.pieces, list.together) * tiles + ceil_div64(ceil_div64(a.rows, per) * tiles, EMBED_WARPS);
    op_launch_next(a.s, dim3((unsigned)blocks), dim3(EMBED_THREADS), SMEM, kernel, (const T*)a.dy, a.dys, list, a.rows, a.n, tiles, per, a.scale, (O*)a.out, a.os);
}
template <typename T, typename O, int VEC>
void embed_rows_pick(const EmbedBackward& a) {
    const int units = (int)ceil_div64(a.n, 32 * VEC);
    if (a.few) {
        op_launch_next(a.s, dim3((unsigned)(a.rows * units)), dim3(EMBED_FEW_WARPS * 32), 0, k_embed_few<T, O, VEC>, a.tokens, (int)a.count, (const T*)a.dy, a.dys, a.n, units, a.scale, (O*)a.out, a.os);
        return;
    }
    // Rows up to 2 KB by loads (125143 tokens evenly over 3640 x 384 fp32: 73 us, by copies 85), rows up to 3 KB by copies of the whole row, longer ones by copies of tiles of 2 KB.  65536 tokens of
    // tables of 73305 and 3640 rows, whole rows of 3 KB and tiles of 2 KB: 640 fp32 111 and 63 us, 119 and 78; 768 fp32 118 and 71, 123 and 76; 1152 bf16 111 and 69, 114 and 72; 1536 bf16 122 and 81, 121 and
    // 79.  Of longer rows, tiles of 3 KB take 16-bit ones no less time and fp32 ones some less, some more: 1024 fp32 182 and 79, by tiles of 2 KB 154 and 80; 1536 fp32 225 and 100, 243 and 115.
    // Rows that start anywhere by loads up to 128 columns, by copies above (3640 x 222: 80 us, by loads 60 where tokens are even and 154 where they are not).
    if constexpr (VEC == 1) {
        if (units == 1) return embed_rows_go<T, O, 1, 1, 8, EmbedLoads>(a);
        if (units == 2) return embed_rows_go<T, O, 1, 2, 8, EmbedLoads>(a);
        if (units <= 4) return embed_rows_go<T, O, 1, 4, 4, EmbedLoads>(a);
        if (units <= 8) return embed_rows_go<T, O, 1, 8, 8, EmbedCopies>(a);
        embed_rows_go<T, O, 1, 16, 4, EmbedCopies>(a);
    } else {
        if (units == 1) return embed_rows_go<T, O, VEC, 1, 8, EmbedLoads>(a);
        if (units <= 4) return embed_rows_go<T, O, VEC, 2, 4, EmbedLoads>(a);
        if (units == 5 || units == 6) return embed_rows_go<T, O, VEC, 6, 4, EmbedCopies>(a);
        embed_rows_go<T, O, VEC, 4, 4, EmbedCopies>(a);
    }
}
template <typename T, int VEC>
void embed_rows_type(const EmbedBackward& a, bool single, bool wide) {
    if (single) return wide ? embed_rows_pick<T, float, VEC>(a) : embed_rows_pick<T, float, 1>(a);
    return wide ? embed_rows_pick<T, T, VEC>(a) : embed_rows_pick<T, T, 1>(a);
}

template <typename T, int VEC>
bool embed_forward_go(cudaStream_t s, const Tokens& tokens, int64_t count, const void* table, int64_t ts, int n, float scale, void* out, int64_t os) {
    const int units = (int)ceil_div64(n, VEC);
#define GO(L, CH, R)                                                                                                                                              \
    do {                                                                                                                                                          \
        const int tiles = (int)ceil_div64(units, (L) * (CH));                                                                                                     \
        const int64_t groups = (count + (R) - 1) / (R), per = EMBED_THREADS / (L), blocks = (groups * tiles + per - 1) / per;                                     \
        if (blocks > INT32_MAX) return false;                                                                                                                     \
        op_launch_next(s, dim3((unsigned)blocks), dim3(EMBED_THREADS), 0, k_embed_forward<T, VEC, L, CH, R>, tokens, count, (const T*)table, ts, n, tiles, scale, (T*)out, os); \
        return true;                                                                                                                                              \
    } while (0)
    if constexpr (VEC == 1) {  // single elements: more of them on their way (146325 x 294 fp16: 114 us with four a lane, 40 with sixteen)
        if (units <= 8) GO(8, 1, 8);
        if (units <= 32) GO(32, 1, 8);
        if (units <= 64) GO(32, 2, 8);
        GO(32, 4, 4);
    }
    if (units <= 8) GO(8, 1, 4);
    if (units <= 32) GO(32, 1, 4);
    if (units <= 64) GO(32, 2, 2);
    GO(32, 4, 1);
#undef GO
}
bool embed_aligned(const void* p, int64_t stride, int size) { return ((uintptr_t)p & 15) == 0 && (stride * size) % 16 == 0; }

int embed_check(int type, int64_t count, int64_t rows, int n, int token_bytes, const void* tokens, char* err, size_t err_len) {
    if (!op_type_size(type)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "type must be TB_TYPE_F32, TB_TYPE_F16 or TB_TYPE_BF16 (got %d)", type);
    if (token_bytes != 4 && token_bytes != 8) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "token_bytes must be 4 or 8 (got %d)", token_bytes);
    if (count < 0 || count > OP_MAX_ENTRIES || rows < 1 || rows > INT32_MAX) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "count must be in [0, 2^31 - 1024] and rows in [1, 2^31)");
    if (n < 1 || n > OP_MAX_COLUMNS) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "n must be in [1, 2^30] (got %d)", n);
    if (count > 0 && !tokens) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_tokens is NULL");
    if ((uintptr_t)tokens % token_bytes) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "tensors must be aligned to their elements");
    return TB_OK;
}

}  // namespace

extern "C" int tb_embedding_forward(const void* d_tokens, int token_bytes, int64_t count, const void* d_table, int64_t table_stride, int type, int64_t rows, int n, float scale, void* d_out,
                                    int64_t out_stride, void* stream, char* err, size_t err_len) {
    if (err && err_len) err[0] = 0;
    const int rc = embed_check(type, count, rows, n, token_bytes, d_tokens, err, err_len), size = op_type_size(type);
    if (rc != TB_OK) return rc;
    if (count == 0) return TB_OK;
    if (!d_table || !d_out) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "a device pointer is NULL");
    if ((rows > 1 && table_stride < n) || (count > 1 && out_stride < n)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "row strides must be at least n");
    if (((uintptr_t)d_table | (uintptr_t)d_out) % size) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "tensors must be aligned to their elements");
    const OpRows outr = {d_out, out_stride * size, count, (int64_t)n * size};
    if (op_extents_meet(outr, {{d_table, table_stride * size, rows, (int64_t)n * size}, op_vector(d_tokens, count, token_bytes)}))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_out overlaps another tensor");
    const bool wide = n % (16 / size) == 0 && embed_aligned(d_table, table_stride, size) && embed_aligned(d_out, out_stride, size);
    const Tokens tokens = {d_tokens, token_bytes == 8, rows};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
#define GO(T, VEC) (wide ? embed_forward_go<T, VEC>(s, tokens, count, d_table, table_stride, n, scale, d_out, out_stride) : embed_forward_go<T, 1>(s, tokens, count, d_table, table_stride, n, scale, d_out, out_stride))
    const bool fits = type == TB_TYPE_F32 ? GO(float, 4) : type == TB_TYPE_F16 ? GO(__half, 8) : GO(__nv_bfloat16, 8);
#undef GO
    if (!fits) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "tokens times columns are too many for one launch");
    return op_launched(err, err_len);
}

extern "C" int64_t tb_embedding_backward_workspace(int64_t count, int64_t rows, int n) {
    EmbedPlan p;
    return embed_plan(count, rows, n, &p) ? embed_bytes(p, n) : TB_ERR_INVALID_ARGUMENT;
}

extern "C" int tb_embedding_backward(const void* d_dy, int64_t dy_stride, int type, const void* d_tokens, int token_bytes, int64_t count, int64_t rows, int n, float scale, void* d_dtable,
                                     int64_t dtable_stride, int dtable_type, void* d_work, int64_t work_bytes, void* stream, char* err, size_t err_len) {
    if (err && err_len) err[0] = 0;
    const int rc = embed_check(type, count, rows, n, token_bytes, d_tokens, err, err_len), size = op_type_size(type);
    if (rc != TB_OK) return rc;
    if (dtable_type != type && dtable_type != TB_TYPE_F32) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "dtable_type must be type or TB_TYPE_F32 (got %d)", dtable_type);
    if (!d_dtable || (count > 0 && !d_dy)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "a device pointer is NULL");
    if ((count > 1 && dy_stride < n) || (rows > 1 && dtable_stride < n)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "row strides must be at least n");
    const int out_size = op_type_size(dtable_type);
    if ((uintptr_t)d_dy % size || (uintptr_t)d_dtable % out_size) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "tensors must be aligned to their elements");
    const OpRows outr = {d_dtable, dtable_stride * out_size, rows, (int64_t)n * out_size};
    if (op_extents_meet(outr, {{d_dy, dy_stride * size, count, (int64_t)n * size}, op_vector(d_tokens, count, token_bytes)}))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_dtable overlaps another tensor");
    EmbedPlan p;
    if (!embed_plan(count, rows, n, &p)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "rows times columns are too many for one launch");
    const int64_t need = embed_bytes(p, n);
    if (need > 0 && (!d_work || work_bytes < need || ((uintptr_t)d_work & 31)))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "the workspace must be aligned and hold %lld bytes (got %lld)", (long long)need, (long long)work_bytes);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const Tokens tokens = {d_tokens, token_bytes == 8, rows};
    int *work = static_cast<int*>(d_work), *total = work + p.words - 1;
    int *key = work + p.words, *id = key + p.list, *key2 = id + p.list, *id2 = key2 + p.list;
    if (!p.few) {
        const int mask = (1 << p.bits) - 1;
        // the counts of the sort by digit k: [k] of as many tables
        const int64_t table = sort_words(p.sort), zeros = p.tables - table + p.done;
        const auto next = [&](int k) { return NextCount{k < p.passes && table ? work + k * table : nullptr, p.sort.keys, SORT_THREADS * p.sort.steps, k * p.bits}; };
        sort_count(s, p.sort, FirstSource{tokens, mask}, count, work, work + table, zeros);
        sort_place(s, p.sort, FirstSource{tokens, mask}, count, work, FirstPut{key, id, total, work + table, zeros, next(1)});
        for (int k = 1; k < p.passes; ++k) {
            sort_place(s, p.sort, NextSource{key, id, total, k * p.bits, mask}, count, work + k * table, NextPut{key2, id2, next(k + 1)});
            std::swap(key, key2);
            std::swap(id, id2);
        }
    }
    float* part = reinterpret_cast<float*>(work + p.words + (p.passes > 1 ? 4 : 2) * p.list);
    const bool wide = n % (16 / size) == 0 && embed_aligned(d_dy, dy_stride, size) && embed_aligned(d_dtable, dtable_stride, out_size);
    const EmbedBackward a = {s, tokens, count, p.few, d_dy, dy_stride, rows, n, scale, d_dtable, dtable_stride, {key, id, total, p.piece, p.pieces, 1, part, work + p.tables}};
    const bool single = dtable_type == TB_TYPE_F32;
    if (type == TB_TYPE_F32) embed_rows_type<float, 4>(a, true, wide);
    else if (type == TB_TYPE_F16) embed_rows_type<__half, 8>(a, single, wide);
    else embed_rows_type<__nv_bfloat16, 8>(a, single, wide);
    return op_launched(err, err_len);
}
