// Rows of a table by token, scaled, and the table's gradient, on the caller's device tensors.
//
//   forward    out[t] = scale * table[token_t]
//   backward   dtable[v] = scale * sum over the tokens t = v of dy[t], every row of the table written once, zeros where no token asks for it
//
// A token outside the table has a row of zeros and no gradient.  Both are bound by memory.  Backward, the tokens are sorted (op_sort.cuh, a stable sort by up
// to ten bits at a time), so that a row's tokens lie together in ascending order.  A warp takes a table row: it finds its tokens in the sorted list
// and adds their rows in registers.  Where that would be a long chain (more than `piece` tokens: a few tokens make up much of any text or board), the list's
// pieces of that many tokens are added up by blocks of their own in the same launch, and a further launch adds up the pieces.  Sums are fp32 in an order that depends
// on the tokens alone, so results repeat bit for bit.
#include "op_sort.cuh"

#include <utility>

namespace {

#define EMBED_THREADS 256
#define EMBED_WARPS 8
#define EMBED_ROWS 8  // table rows per warp at most

struct Tokens {
    const void* p;
    int wide;  // 64-bit ones
    int64_t rows;
    // -1 where the table has no such row
    __device__ __forceinline__ int operator()(int64_t i) const {
        const int64_t t = wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int*>(p)[i];
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
    int *key, *id, *count;  // count: of the tokens in the table, and (zero here) of the long lists
    NextCount next;
    __device__ __forceinline__ void operator()(int64_t i, int v, int place) const {
        if (place < 0) return;
        key[place] = v;
        id[place] = (int)i;
        next(v, place);
    }
    __device__ __forceinline__ void rest(const int*, const int* begin, const SortPlan& p) const {
        if (blockIdx.x == 0 && threadIdx.x == 0) count[0] = begin[p.keys], count[1] = 0;
    }
};
// further digits, of what the digits before have sorted
struct NextSource {
    const int *sorted, *count;
    int shift, mask;
    __device__ __forceinline__ int operator()(int64_t i) const {
        const int v = sorted[i];  // behind the last one anything
        return i < *count ? v : -1;
    }
    __device__ __forceinline__ int key(int v) const { return v < 0 ? -1 : v >> shift & mask; }
};
struct NextPut {
    const int* id_in;
    int *key, *id;
    NextCount next;
    __device__ __forceinline__ void operator()(int64_t i, int v, int place) const {
        if (place < 0) return;
        key[place] = v;
        id[place] = id_in[i];
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

template <typename T, int VEC, int CH>
__device__ __forceinline__ void embed_load(OpRaw<T, VEC> (&x)[CH], const T* dy, int64_t dy_stride, int row, bool there, int first, int n) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = first + c * 32 * VEC;
        x[c].zero();
        if (there && col < n) x[c].load(dy + row * dy_stride + col);
    }
}
template <typename T, int VEC, int CH>
__device__ __forceinline__ void embed_add(float (&acc)[CH][VEC], const OpRaw<T, VEC> (&x)[CH]) {
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[c][i] += x[c].get(i);
}
template <int VEC, int CH>
__device__ __forceinline__ void embed_zero(float (&acc)[CH][VEC]) {
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[c][i] = 0.0f;
}

struct EmbedLong {       // a token whose list is longer than a piece: its first sum, and the list's last piece
    int token, first, last;
};
struct EmbedList {
    const int *key, *id;
    int* count;          // of the tokens in the table, and of the long lists
    int piece, pieces;   // tokens to a piece, and how many pieces there can be
    EmbedLong* lists;    // the long ones in any order
    float* part;         // [pieces][2][n]: the sums of a piece's first and of its last token, where those have long lists
};

// Blocks below pieces * tiles: a piece of the list and a tile of columns.  The others: `per` table rows and a tile per warp; it looks for the first row's place in the
// list once and reads on from there, 32 entries at a time.
template <typename T, typename O, int VEC, int CH>
__global__ void __launch_bounds__(EMBED_THREADS, 4)
k_embed_rows(const T* dy, int64_t dy_stride, EmbedList list, int64_t rows, int n, int tiles, int per, float scale, O* __restrict__ out, int64_t out_stride) {
    constexpr int TILE = 32 * VEC * CH, U = CH == 1 ? 8 : CH == 2 ? 4 : 2;  // rows on their way together
    __shared__ float s_part[EMBED_WARPS][TILE];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, piece_blocks = list.pieces * tiles;
    op_next_may_start();
    op_wait_for_previous();
    const int count = *list.count;
    float acc[CH][VEC];
    if ((int64_t)blockIdx.x >= piece_blocks) {
        const int64_t unit = ((int64_t)blockIdx.x - piece_blocks) * EMBED_WARPS + warp, group = unit / tiles, row0 = group * per;
        if (row0 >= rows) return;
        const int first = ((int)(unit - group * tiles) * 32 * CH + lane) * VEC, many = (int)min((int64_t)per, rows - row0);
        const int end_row = (int)row0 + many;
        const auto store = [&](int64_t v) {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int col = first + c * 32 * VEC;
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[c][i] *= scale;
                if (col < n) embed_store<O, VEC>(out + v * out_stride + col, acc[c]);
            }
            embed_zero(acc);
        };
        int v = (int)row0, last = -1;  // acc is v's; the key before the window
        embed_zero(acc);
        for (int at = embed_below(list.key, 0, count, v, lane);;) {
            const int key = lane < count - at ? list.key[at + lane] : INT32_MAX, id = lane < count - at ? list.id[at + lane] : 0;
            const int ahead = list.piece < count - at - lane ? list.key[at + list.piece + lane] : -1, before = __shfl_up_sync(0xffffffffu, key, 1);
            // up to the window's first list that is longer than a piece, which is added up by pieces
            const unsigned longer = __ballot_sync(0xffffffffu, ahead == key && key != (lane ? before : last) && key < end_row);
            const int mine = __popc(__ballot_sync(0xffffffffu, key < end_row)), here = longer ? __ffs(longer) - 1 : mine;
            for (int j0 = 0; j0 < here; j0 += U) {
                OpRaw<T, VEC> x[U][CH];
#pragma unroll
                for (int u = 0; u < U; ++u) embed_load<T, VEC, CH>(x[u], dy, dy_stride, __shfl_sync(0xffffffffu, id, j0 + u), j0 + u < here, first, n);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int k = __shfl_sync(0xffffffffu, key, j0 + u);
                    if (j0 + u >= here) break;
                    for (; v < k; ++v) store(v);
                    embed_add(acc, x[u]);
                }
            }
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
        return;
    }
    const int piece = blockIdx.x / tiles, tile = blockIdx.x - piece * tiles, first = (tile * 32 * CH + lane) * VEC;
    if ((int64_t)piece * list.piece >= count) return;
    const int from = piece * list.piece, to = list.piece < count - from ? from + list.piece : count, first_key = list.key[from], last_key = list.key[to - 1];
    for (int slot = 0; slot < (first_key == last_key ? 1 : 2); ++slot) {
        // the token's entries of this piece, and whether the list is longer than a piece
        const int v = slot ? last_key : first_key;
        const int b = slot ? embed_below(list.key, from, to, v, lane) : from, e = slot || last_key == v ? to : embed_below(list.key, from, to, v + 1, lane);
        const bool begins = slot || from == 0 || list.key[from - 1] != v;
        const bool longer = begins ? list.piece < count - b && list.key[b + list.piece] == v : e - from == list.piece || list.key[e - 1 - list.piece] == v;
        if (!longer) continue;
        if (begins && tile == 0 && warp == 0) {
            const int end = embed_below(list.key, to, count, v + 1, lane);
            if (lane == 0) list.lists[atomicAdd(list.count + 1, 1)] = {v, piece * 2 + slot, (end - 1) / list.piece};
        }
        const int share = (e - b + EMBED_WARPS - 1) / EMBED_WARPS;
        embed_zero(acc);
        const int mine_to = min(b + (warp + 1) * share, e);
        for (int i0 = b + warp * share; i0 < mine_to; i0 += 32) {
            const int many = min(32, mine_to - i0), id = lane < many ? list.id[i0 + lane] : 0;
            for (int j0 = 0; j0 < many; j0 += U) {
                OpRaw<T, VEC> x[U][CH];
#pragma unroll
                for (int u = 0; u < U; ++u) embed_load<T, VEC, CH>(x[u], dy, dy_stride, __shfl_sync(0xffffffffu, id, j0 + u), j0 + u < many, first, n);
#pragma unroll
                for (int u = 0; u < U; ++u) embed_add(acc, x[u]);
            }
        }
        __syncthreads();  // the sums of the slot before are read
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < VEC; ++i) s_part[warp][(c * VEC + i) * 32 + lane] = acc[c][i];
        __syncthreads();
        for (int at = threadIdx.x; at < TILE; at += EMBED_THREADS) {
            float sum = s_part[0][at];
#pragma unroll
            for (int w = 1; w < EMBED_WARPS; ++w) sum += s_part[w][at];
            const int col = ((tile * CH + at / 32 / VEC) * 32 + at % 32) * VEC + at / 32 % VEC;
            if (col < n) list.part[((int64_t)piece * 2 + slot) * n + col] = sum;
        }
    }
}

// The rows with long lists, 32 columns at a time: a warp adds up a list's pieces, or a block's warps a share of them each where they are more than EMBED_ALONE.
#define EMBED_ALONE 32
template <int U>
__device__ __forceinline__ float embed_pieces(const EmbedList& list, const EmbedLong& l, int from, int to, int col, int n) {
    float sum = 0.0f;
    for (int p0 = from; p0 < to; p0 += U) {
        float t[U];
#pragma unroll
        for (int i = 0; i < U; ++i) t[i] = p0 + i < to && col < n ? list.part[(int64_t)(p0 + i == 0 ? l.first : (l.first / 2 + p0 + i) * 2) * n + col] : 0.0f;
#pragma unroll
        for (int i = 0; i < U; ++i) sum += t[i];
    }
    return sum;
}
template <typename O>
__global__ void __launch_bounds__(EMBED_THREADS)
k_embed_join(EmbedList list, int n, int tiles, float scale, O* __restrict__ out, int64_t out_stride) {
    __shared__ float s_part[EMBED_WARPS][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    op_next_may_start();
    op_wait_for_previous();
    const int64_t items = (int64_t)list.count[1] * tiles;
    for (int64_t item = (int64_t)blockIdx.x * EMBED_WARPS + warp; item < items; item += (int64_t)gridDim.x * EMBED_WARPS) {
        const EmbedLong l = list.lists[item / tiles];
        const int col = (int)(item % tiles) * 32 + lane, sums = l.last - l.first / 2 + 1;
        if (sums > EMBED_ALONE) continue;
        const float sum = embed_pieces<8>(list, l, 0, sums, col, n);
        if (col < n) out[(int64_t)l.token * out_stride + col] = op_round<O>(sum * scale);
    }
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const EmbedLong l = list.lists[item / tiles];
        const int col = (int)(item % tiles) * 32 + lane, sums = l.last - l.first / 2 + 1, share = (sums + EMBED_WARPS - 1) / EMBED_WARPS;
        if (sums <= EMBED_ALONE) continue;
        s_part[warp][lane] = embed_pieces<16>(list, l, warp * share, min((warp + 1) * share, sums), col, n);
        __syncthreads();
        if (warp == 0 && col < n) {
            float sum = s_part[0][lane];
#pragma unroll
            for (int w = 1; w < EMBED_WARPS; ++w) sum += s_part[w][lane];
            out[(int64_t)l.token * out_stride + col] = op_round<O>(sum * scale);
        }
        __syncthreads();
    }
}

// ---- plans -------------------------------------------------------------------------------------------------------------------
struct EmbedPlan {
    int passes, bits;    // of the sort
    SortPlan sort;
    int piece, pieces;
    int64_t words, list; // 32-bit ones of the sort's workspace and the counts, of each sorted list; then the long lists and the pieces' sums
};
bool embed_plan(int64_t count, int64_t rows, int n, EmbedPlan* p) {
    if (count < 0 || count > OP_MAX_ENTRIES || rows < 1 || rows > INT32_MAX || n < 1 || n > OP_MAX_COLUMNS) return false;
    int bits = 1;
    while (((int64_t)1 << bits) < rows) ++bits;
    p->passes = (bits + 9) / 10;
    p->bits = (bits + p->passes - 1) / p->passes;
    p->sort = sort_plan(count, 1 << p->bits, 1);
    // pieces of 32 tokens, or more where there were over 2048 of them: their sums are one chain per warp when they are joined
    p->piece = 32;
    while (count > (int64_t)p->piece * 2048) p->piece *= 2;
    p->pieces = (int)((count + p->piece - 1) / p->piece);
    p->words = (p->passes * sort_words(p->sort) + 2 + 7) / 8 * 8;
    p->list = (count + 7) / 8 * 8;
    // what one launch takes; tensors that fit a GPU are far below
    return (p->pieces + rows / EMBED_WARPS + 2) * ceil_div64(n, 32) <= INT32_MAX;
}
int64_t embed_lists(const EmbedPlan& p) { return ((int64_t)p.pieces * 3 + 7) / 8 * 8; }
int64_t embed_bytes(const EmbedPlan& p, int n) { return 4 * (p.words + (p.passes > 1 ? 4 : 2) * p.list + embed_lists(p) + (int64_t)p.pieces * 2 * n); }

struct EmbedBackward {
    cudaStream_t s;
    const void* dy;
    int64_t dys, rows;
    int n;
    float scale;
    void* out;
    int64_t os;
    EmbedList list;
};
template <typename T, typename O, int VEC, int CH>
void embed_rows_go(const EmbedBackward& a) {
    const int tiles = (int)ceil_div64(a.n, 32 * VEC * CH);
    // several rows per warp where that leaves every SM's 32 warps a few turns: they share the search
    const int64_t turns = a.rows * tiles / ((int64_t)sm_count() * 128);
    const int per = (int)(turns < 1 ? 1 : turns > EMBED_ROWS ? EMBED_ROWS : turns);
    const int64_t blocks = (int64_t)a.list.pieces * tiles + ceil_div64(ceil_div64(a.rows, per) * tiles, EMBED_WARPS);
    op_launch_next(a.s, dim3((unsigned)blocks), dim3(EMBED_THREADS), 0, k_embed_rows<T, O, VEC, CH>, (const T*)a.dy, a.dys, a.list, a.rows, a.n, tiles, per, a.scale, (O*)a.out, a.os);
    if (a.list.pieces > 1) {
        const int columns = (int)ceil_div64(a.n, 32);
        const int64_t items = (int64_t)a.list.pieces * columns, most = 8 * (int64_t)sm_count();
        op_launch_next(a.s, dim3((unsigned)(items < most ? items : most)), dim3(EMBED_THREADS), 0, k_embed_join<O>, a.list, a.n, columns, a.scale, (O*)a.out, a.os);
    }
}
template <typename T, typename O, int VEC>
void embed_rows_pick(const EmbedBackward& a) {
    // up to sixteen columns a lane (more do not fit 64 registers with the rows on their way); three accesses where they leave no more lanes without a column than two
    const int units = (int)ceil_div64(a.n, 32 * VEC);
    if (units == 1) return embed_rows_go<T, O, VEC, 1>(a);
    if constexpr (VEC < 8)
        if (ceil_div(units, 3) * 3 <= ceil_div(units, 2) * 2) return embed_rows_go<T, O, VEC, 3>(a);
    embed_rows_go<T, O, VEC, 2>(a);
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
    if (count < 0 || count > OP_MAX_ENTRIES || rows < 1 || rows > INT32_MAX) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "count must be in [0, 2^31) and rows in [1, 2^31)");
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
    if (!d_work || work_bytes < need || ((uintptr_t)d_work & 31))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "the workspace must be aligned and hold %lld bytes (got %lld)", (long long)need, (long long)work_bytes);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    int *work = static_cast<int*>(d_work), *total = work + p.words - 2;
    int *key = work + p.words, *id = key + p.list, *key2 = id + p.list, *id2 = key2 + p.list;
    const Tokens tokens = {d_tokens, token_bytes == 8, rows};
    const int mask = (1 << p.bits) - 1;
    // the counts of the sort by digit k: [k] of as many tables
    const int64_t table = sort_words(p.sort);
    const auto next = [&](int k) { return NextCount{k < p.passes && table ? work + k * table : nullptr, p.sort.keys, SORT_THREADS * p.sort.steps, k * p.bits}; };
    sort_count(s, p.sort, FirstSource{tokens, mask}, count, work, work + table, (p.passes - 1) * table);
    sort_place(s, p.sort, FirstSource{tokens, mask}, count, work, FirstPut{key, id, total, next(1)});
    for (int k = 1; k < p.passes; ++k) {
        sort_place(s, p.sort, NextSource{key, total, k * p.bits, mask}, count, work + k * table, NextPut{id, key2, id2, next(k + 1)});
        std::swap(key, key2);
        std::swap(id, id2);
    }
    int* lists = work + p.words + (p.passes > 1 ? 4 : 2) * p.list;
    const bool wide = n % (16 / size) == 0 && embed_aligned(d_dy, dy_stride, size) && embed_aligned(d_dtable, dtable_stride, out_size);
    const EmbedBackward a = {s, d_dy, dy_stride, rows, n, scale, d_dtable, dtable_stride, {key, id, total, p.piece, p.pieces, reinterpret_cast<EmbedLong*>(lists), reinterpret_cast<float*>(lists + embed_lists(p))}};
    const bool single = dtable_type == TB_TYPE_F32;
    if (type == TB_TYPE_F32) embed_rows_type<float, 4>(a, true, wide);
    else if (type == TB_TYPE_F16) embed_rows_type<__half, 8>(a, single, wide);
    else embed_rows_type<__nv_bfloat16, 8>(a, single, wide);
    return op_launched(err, err_len);
}
