// draft_tree.hip -- what surrounds the attention of drafted tokens (tree_attn.hip) on the device, so that a speculative step
// needs no host round trip: block tables and slot maps from request lengths, the accepted path of a tree, and the move of the
// accepted keys and values to the end of the history.  All integer work and copies: results are exact and do not depend on
// the order in which workgroups run.
#include "kernels.h"

namespace mi355q
{
namespace
{

// ---------------------------------------------------------------------------------------------- block tables
// Every request holds block_counts[b] blocks; past + new tokens need ceil((past + new) / tokens_per_block).  The missing
// ones come from the front of a ring of free block indices, in request order; a request that ends returns its blocks to
// the ring's back.  Two launches: the plan (prefix sums over the requests, one workgroup) and the fill (tables, ring,
// pointers of every pool, slots).  The fill reads no table or ring entry that it writes, and the state only through the
// plan's records, so updating it in place is safe.
// 256 requests of 512 blocks in 64 pools: plan 3.6 us, fill 21.4 us for the 134 MB of pointers = 6.3 TB/s (a plain fill: 6.9); 8 requests
// of 64 in 32 pools: 2.6 + 2.8 us, two launches.  One launch with the sums in every workgroup would read all requests in each.
struct TableArgs
{
    const int32_t* past_lengths;
    const int32_t* new_lengths;
    int32_t* block_table;
    const int32_t* block_counts;
    int32_t* block_counts_out;
    int32_t* free_blocks;
    const int32_t* free_state;
    int32_t* free_state_out;
    const int64_t* pool_bases;
    int64_t* block_pointers;
    int32_t* token_offsets;
    int64_t* slot_map;
    int32_t* status;
    int4* rows; // workspace [batch]: blocks held before, blocks granted (-1: released), first ring position, status
    int64_t block_bytes;
    int batch, max_blocks, num_blocks, num_pools, num_tokens, tpb, tpb_log2;
    int pools_per_wg, planes, wgs_per_row;
};

constexpr int PLAN_THREADS = 1024;

// exclusive prefix sums of NV values over the workgroup; sum receives the totals
template <int NV>
__device__ __forceinline__ void exclusive_scan(const int64_t (&v)[NV], int64_t (&before)[NV], int64_t (&sum)[NV], int64_t (*lds)[PLAN_THREADS / 64])
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t x[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i)
        x[i] = v[i];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1)
#pragma unroll
        for (int i = 0; i < NV; ++i)
        {
            const int64_t y = __shfl_up(x[i], o);
            x[i] += lane >= o ? y : 0;
        }
    __syncthreads(); // the previous sums have been read
    if (lane == 63)
#pragma unroll
        for (int i = 0; i < NV; ++i)
            lds[i][wave] = x[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i)
    {
        before[i] = x[i] - v[i];
        sum[i] = 0;
        for (int w = 0; w < (int) blockDim.x / 64; ++w)
        {
            before[i] += w < wave ? lds[i][w] : 0;
            sum[i] += lds[i][w];
        }
    }
}

// x mod N for 0 <= x < 3 N (a 64-bit remainder is over a hundred instructions)
__device__ __forceinline__ int wrap(int64_t x, int64_t N)
{
    x = x >= N ? x - N : x;
    return (int) (x >= N ? x - N : x);
}

// one workgroup of up to 1024 threads
__global__ __launch_bounds__(PLAN_THREADS) void table_plan_kernel(TableArgs p)
{
    __shared__ int64_t lds[3][PLAN_THREADS / 64];
    const int64_t N = p.num_blocks;
    const int head = p.free_state[0] >= 0 && p.free_state[0] < N ? p.free_state[0] : 0;
    const int64_t avail = min((int64_t) max(p.free_state[1], 0), N);
    int64_t demand = 0, granted = 0, returned = 0, tokens = 0;
    for (int b0 = 0; b0 < p.batch; b0 += blockDim.x)
    {
        const int b = b0 + threadIdx.x;
        int count = 0, status = 0;
        int64_t v[3] = {0, 0, 0}; // blocks asked for, blocks returned, tokens
        bool release = false;
        if (b < p.batch)
        {
            const int64_t past = p.past_lengths[b], add = p.new_lengths[b];
            count = p.block_counts[b];
            release = add < 0;
            v[2] = max(add, (int64_t) 0);
            if (past < 0 || count < 0 || count > p.max_blocks || count > N)
                status = 3;
            else if (release)
                v[1] = count;
            else
            {
                const int64_t total = (past + add + p.tpb - 1) >> p.tpb_log2;
                if (total > p.max_blocks)
                    status = 2;
                else
                    v[0] = max(total - count, (int64_t) 0);
            }
        }
        int64_t before[3], sum[3];
        exclusive_scan(v, before, sum, lds);
        // first come, first served: a request that the blocks do not reach for gets none, nor does any behind it that asks.
        // So what is granted is the demand up to the first one refused
        const int64_t from_need = demand + before[0];
        int64_t need = v[0];
        if (need > 0 && from_need + need > avail)
        {
            status = 1;
            need = 0;
        }
        const int64_t mine[1] = {need};
        int64_t unused[1], grant[1];
        if (demand + sum[0] > avail) // uniform
            exclusive_scan(mine, unused, grant, lds);
        else
            grant[0] = sum[0];
        if (b < p.batch)
        {
            const bool gives = release && status == 0;
            // ring positions of granted blocks end before the free ones do, those of returned blocks (more than N in all only
            // with a corrupt state) behind them
            const int64_t from = gives ? avail + min(returned + before[1], N) : min(from_need, N);
            p.rows[b] = make_int4(count, gives ? -1 : (int) need, wrap(head + from, N), status);
            p.token_offsets[b] = (int) min(tokens + before[2], (int64_t) INT32_MAX);
            p.status[b] = status;
            p.block_counts_out[b] = gives ? 0 : count + (int) need;
        }
        demand += sum[0];
        returned += sum[1];
        tokens += sum[2];
        granted += grant[0];
    }
    __syncthreads(); // free_state has been read by everyone
    if (threadIdx.x == 0)
    {
        p.token_offsets[p.batch] = (int) min(tokens, (int64_t) INT32_MAX);
        p.free_state_out[0] = wrap(head + granted, N);
        p.free_state_out[1] = (int) min(avail - granted + returned, N);
    }
}

// the index of block j of a request, from the table or, for a block granted in this call, from the ring; -1: none
__device__ __forceinline__ int block_index(const TableArgs& p, int b, const int4& row, int j)
{
    int idx = -1;
    if (row.y >= 0 && row.x >= 0 && row.x <= p.max_blocks && j < row.x + row.y)
        idx = j < row.x ? p.block_table[(size_t) b * p.max_blocks + j]
                        : p.free_blocks[wrap((int64_t) row.z + j - row.x, p.num_blocks)];
    return idx >= 0 && idx < p.num_blocks ? idx : -1;
}

// the slot of new token t: its request by bisection of the offsets
__device__ __forceinline__ void write_slot(const TableArgs& p, int t)
{
    int64_t slot = -1;
    if (t < p.token_offsets[p.batch])
    {
        int lo = 0, hi = p.batch; // the last request whose first token is <= t and that has tokens
        while (hi - lo > 1)
        {
            const int mid = (lo + hi) >> 1;
            if (p.token_offsets[mid] <= t)
                lo = mid;
            else
                hi = mid;
        }
        const int4 row = p.rows[lo];
        if (row.w == 0)
        {
            const int64_t pos = (int64_t) p.past_lengths[lo] + (t - p.token_offsets[lo]);
            const int idx = block_index(p, lo, row, (int) (pos >> p.tpb_log2));
            if (idx >= 0)
                slot = ((int64_t) idx << p.tpb_log2) + (pos & (p.tpb - 1));
        }
    }
    p.slot_map[t] = slot;
}

// grid: a 1-D list of workgroups of 256 threads, first (ceil(max_blocks / 512), batch, pool groups + 1) of them with two blocks of
// the table per thread (the last pool group does the table and the ring), then those of the slots, one token per thread.
// Bound by the pointer stores.
template <bool PAIRS>
__global__ __launch_bounds__(256) void table_fill_kernel(TableArgs p)
{
    const uint32_t per_plane = p.wgs_per_row * p.batch, plane = blockIdx.x / per_plane, in_plane = blockIdx.x % per_plane;
    if ((int) plane > p.planes)
    {
        const int64_t t = ((int64_t) blockIdx.x - (int64_t) per_plane * (p.planes + 1)) * 256 + threadIdx.x;
        if (t < p.num_tokens)
            write_slot(p, (int) t);
        return;
    }
    const int b = in_plane / p.wgs_per_row, j = 2 * (in_plane % p.wgs_per_row * 256 + threadIdx.x);
    if (j >= p.max_blocks)
        return;
    const int4 row = p.rows[b];
    if ((int) plane == p.planes)
    {
        for (int k = j; k < min(j + 2, p.max_blocks); ++k)
        {
            int32_t* entry = p.block_table + (size_t) b * p.max_blocks + k;
            if (row.y < 0 && k < row.x) // released
                p.free_blocks[wrap((int64_t) row.z + k, p.num_blocks)] = *entry;
            else if (row.y > 0 && k >= row.x && k < row.x + row.y) // granted
                *entry = p.free_blocks[wrap((int64_t) row.z + k - row.x, p.num_blocks)];
        }
        return;
    }
    const int i0 = block_index(p, b, row, j), i1 = j + 1 < p.max_blocks ? block_index(p, b, row, j + 1) : -1;
    const int64_t k0 = i0 * p.block_bytes, k1 = i1 * p.block_bytes, v = p.num_blocks * p.block_bytes;
    const int lo = plane * p.pools_per_wg, hi = min(lo + p.pools_per_wg, p.num_pools);
    for (int pool = lo; pool < hi; ++pool)
    {
        const int64_t base = p.pool_bases[pool];
        int64_t* out = p.block_pointers + (((size_t) pool * p.batch + b) * 2) * p.max_blocks + j;
        const longlong2 kk = make_longlong2(i0 < 0 ? 0 : base + k0, i1 < 0 ? 0 : base + k1);
        const longlong2 vv = make_longlong2(i0 < 0 ? 0 : base + k0 + v, i1 < 0 ? 0 : base + k1 + v);
        if constexpr (PAIRS)
        {
            *reinterpret_cast<longlong2*>(out) = kk;
            *reinterpret_cast<longlong2*>(out + p.max_blocks) = vv;
        }
        else
        {
            out[0] = kk.x;
            out[p.max_blocks] = vv.x;
            if (j + 1 < p.max_blocks)
            {
                out[1] = kk.y;
                out[p.max_blocks + 1] = vv.y;
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------- accepted path
// One wave per sequence walks its tree from node 0: from node c it goes to the lowest child (parent c, index > c) whose drafted
// token is the model's token after c.  The nodes sit in registers, 4 per lane (256 nodes; larger trees re-read memory): a step
// is a compare, a ballot and a lane read, so the call costs one round trip to memory and a launch: one tree of 27 nodes 3.1 us, 512
// of 64 nodes 5.8 us.
__global__ __launch_bounds__(256) void tree_accept_kernel(const int32_t* draft_tokens, const int32_t* parents,
    const int32_t* target_tokens, const int32_t* draft_offsets, int32_t* accept_path, int32_t* accept_counts,
    int32_t* accepted_tokens, int batch, int num_tokens, int max_path)
{
    const int lane = threadIdx.x & 63;
    const int b = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (b >= batch)
        return;
    const int off = draft_offsets[b];
    const int64_t n64 = (int64_t) draft_offsets[b + 1] - off;
    const int n = off >= 0 && n64 > 0 && off + n64 <= num_tokens ? (int) n64 : 0;
    constexpr int R = 4;
    int tok[R], par[R], tgt[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
    {
        const int i = lane + 64 * r;
        const bool in = i < n;
        tok[r] = in ? draft_tokens[off + i] : 0;
        par[r] = in ? parents[off + i] : -1;
        tgt[r] = in ? target_tokens[off + i] : 0;
    }
    int32_t* path = accept_path + (size_t) b * max_path;
    int32_t* said = accepted_tokens + (size_t) b * max_path;
    int cur = n > 0 ? 0 : -1, count = 0;
    while (cur >= 0 && count < max_path)
    {
        int want = 0;
        if (cur < 64 * R)
        {
#pragma unroll
            for (int r = 0; r < R; ++r)
                want = cur >> 6 == r ? __builtin_amdgcn_readlane(tgt[r], cur & 63) : want;
        }
        else
            want = target_tokens[off + cur];
        if (lane == 0)
        {
            path[count] = cur;
            said[count] = want;
        }
        ++count;
        int next = -1;
#pragma unroll
        for (int r = 0; r < R; ++r)
        {
            const int i = lane + 64 * r;
            const uint64_t hit = __ballot(i < n && i > cur && par[r] == cur && tok[r] == want);
            if (next < 0 && hit)
                next = 64 * r + __builtin_ctzll(hit);
        }
        for (int i0 = 64 * R; next < 0 && i0 < n; i0 += 64)
        {
            const int i = i0 + lane;
            const uint64_t hit = __ballot(i < n && i > cur && parents[off + min(i, n - 1)] == cur && draft_tokens[off + min(i, n - 1)] == want);
            if (hit)
                next = i0 + __builtin_ctzll(hit);
        }
        cur = __builtin_amdgcn_readfirstlane(next);
    }
    for (int i = count + lane; i < max_path; i += 64)
    {
        path[i] = -1;
        said[i] = -1;
    }
    if (lane == 0)
        accept_counts[b] = count;
}

// ---------------------------------------------------------------------------------------------- commit
// Slot past + i of every pool takes the keys and values of slot past + path[i].  In place: paths rise strictly (a parent's
// index is below its children's), so slot past + i is never a source of a later entry, and a thread owns the same bytes
// of a row for all entries: it loads 8 entries, then stores them.
// grid (batch, pools), 256 threads over K / V x heads x row chunks.  One wave reads the path, checks it and finds the rows'
// addresses, 64 entries at a time, all of a lane's loads side by side: what bounds the call is that chain of three round trips
// (lengths and path, block pointers, rows), then the rows it moves: 32 layers of 8 heads of 128, one sequence 3.8 us, 32 sequences 8.4 us
// for 25 MB.  Every thread following the path by itself took 15.2 us for those.
typedef __attribute__((ext_vector_type(4))) uint32_t commit_vec16;
typedef __attribute__((ext_vector_type(2))) uint32_t commit_vec8;
template <typename V>
__global__ __launch_bounds__(256) void commit_path_kernel(const int64_t* block_pointers, const int32_t* past_lengths,
    const int32_t* accept_path, const int32_t* accept_counts, int32_t* new_lengths, int batch, int max_blocks, int tpb_log2,
    int num_kv_heads, int row_bytes, int max_path)
{
    constexpr int C = 64, E = 8; // entries per pass of the wave, per round of loads and stores
    __shared__ int64_t src[2][C], dst[2][C];
    __shared__ int refused;
    const int b = blockIdx.x, pool = blockIdx.y, tid = threadIdx.x;
    const int past = past_lengths[b], given = accept_counts[b];
    const int32_t* path = accept_path + (size_t) b * max_path;
    const int64_t* kp = block_pointers + ((size_t) pool * batch + b) * 2 * max_blocks;
    const int count = min(given, max_path);
    const int tpb_mask = (1 << tpb_log2) - 1;
    // entries c0 .. c0 + 63: their addresses into src / dst; true if one of them cannot be moved
    auto find = [&](int c0)
    {
        const int i = c0 + tid, node = path[min(i, max_path - 1)], before = i > 0 ? path[min(i, max_path) - 1] : -1;
        bool bad = past < 0 || given < 0;
        if (!bad && i < count)
        {
            const int64_t s = (int64_t) past + node, d = (int64_t) past + i;
            bad = node <= before || (s >> tpb_log2) >= max_blocks; // (rising from 0 on: d <= s)
            if (!bad)
            {
                const int64_t ks = kp[s >> tpb_log2], vs = kp[max_blocks + (s >> tpb_log2)];
                const int64_t kd = kp[d >> tpb_log2], vd = kp[max_blocks + (d >> tpb_log2)];
                bad = ks == 0 || vs == 0 || kd == 0 || vd == 0;
                src[0][tid] = ks + (s & tpb_mask) * row_bytes;
                src[1][tid] = vs + (s & tpb_mask) * row_bytes;
                dst[0][tid] = kd + (d & tpb_mask) * row_bytes;
                dst[1][tid] = vd + (d & tpb_mask) * row_bytes;
            }
        }
        return __any(bad);
    };
    if (tid < 64)
    {
        bool bad = false;
        // the first entries last: their addresses stay
        for (int c0 = count > C ? (count - 1) / C * C : 0; c0 >= 0; c0 -= C)
            bad |= find(c0);
        if (tid == 0)
        {
            refused = bad;
            if (pool == 0)
                new_lengths[b] = bad ? past : past + count;
        }
    }
    __syncthreads();
    if (refused)
        return;
    const int chunks = row_bytes / (int) sizeof(V), work = 2 * num_kv_heads * chunks;
    for (int c0 = 0; c0 < count; c0 += C)
    {
        if (c0 > 0)
        {
            __syncthreads(); // the addresses before have been read
            if (tid < 64)
                find(c0);
            __syncthreads();
        }
        const int here = min(count - c0, C);
        for (int w = tid; w < work; w += 256)
        {
            const int kv = w / (num_kv_heads * chunks), hc = w % (num_kv_heads * chunks), h = hc / chunks, c = hc % chunks;
            const int64_t at = ((int64_t) h << tpb_log2) * row_bytes + (int64_t) c * sizeof(V);
            typedef __attribute__((address_space(1))) V global_v;
            for (int i0 = 0; i0 < here; i0 += E)
            {
                V x[E];
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (i0 + e < here && src[kv][i0 + e] != dst[kv][i0 + e])
                        x[e] = *(const global_v*) (src[kv][i0 + e] + at);
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (i0 + e < here && src[kv][i0 + e] != dst[kv][i0 + e])
                        *(global_v*) (dst[kv][i0 + e] + at) = x[e];
            }
        }
    }
}

int log2_exact(int v, const char* what)
{
    MQ_CHECK(v > 0 && (v & (v - 1)) == 0 && v <= (1 << 20), "%s must be a power of 2, got %d", what, v);
    int l = 0;
    while ((1 << l) < v)
        ++l;
    return l;
}

// do [a, a + an) and [b, b + bn) share a byte
bool overlap(const void* a, size_t an, const void* b, size_t bn)
{
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && x < y + bn && y < x + an;
}
} // namespace

size_t kv_block_tables_workspace_size(int batch)
{
    MQ_CHECK(batch >= 0 && batch <= 65535, "batch %d", batch);
    return (size_t) batch * sizeof(int4);
}

void kv_block_tables(const mi355q_kv_block_tables_params& q, hipStream_t stream)
{
    MQ_CHECK(q.batch >= 0 && q.batch <= 65535, "batch %d", q.batch);
    MQ_CHECK(q.max_blocks_per_seq > 0 && q.max_blocks_per_seq <= (1 << 24), "max_blocks_per_seq %d", q.max_blocks_per_seq);
    MQ_CHECK(q.num_blocks > 0 && q.num_pools >= 0 && q.num_tokens >= 0, "num_blocks %d, num_pools %d, num_tokens %d", q.num_blocks,
        q.num_pools, q.num_tokens);
    MQ_CHECK(q.block_bytes > 0, "block_bytes %lld", (long long) q.block_bytes);
    TableArgs a{};
    a.tpb_log2 = log2_exact(q.tokens_per_block, "tokens_per_block");
    if (q.batch == 0)
        return;
    MQ_CHECK(q.past_lengths && q.new_lengths && q.block_table && q.block_counts && q.block_counts_out && q.free_blocks && q.free_state
            && q.free_state_out && q.token_offsets && q.status,
        "null tensor");
    MQ_CHECK(q.num_pools == 0 || (q.pool_bases && q.block_pointers), "null pool_bases / block_pointers");
    MQ_CHECK(q.num_tokens == 0 || q.slot_map, "null slot_map");
    MQ_CHECK(q.workspace && q.workspace_bytes >= kv_block_tables_workspace_size(q.batch) && (reinterpret_cast<uintptr_t>(q.workspace) & 15) == 0,
        "workspace too small: %zu < %zu (or not 16-byte aligned)", q.workspace_bytes, kv_block_tables_workspace_size(q.batch));
    const size_t rows = (size_t) q.batch * sizeof(int32_t);
    MQ_CHECK(!overlap(q.past_lengths, rows, q.block_counts_out, rows) && !overlap(q.past_lengths, rows, q.token_offsets, rows + 4)
            && !overlap(q.past_lengths, rows, q.status, rows),
        "past_lengths overlaps an output");
    MQ_CHECK(q.block_counts == q.block_counts_out || !overlap(q.block_counts, rows, q.block_counts_out, rows),
        "block_counts_out overlaps block_counts without being it");
    a.past_lengths = q.past_lengths;
    a.new_lengths = q.new_lengths;
    a.block_table = q.block_table;
    a.block_counts = q.block_counts;
    a.block_counts_out = q.block_counts_out;
    a.free_blocks = q.free_blocks;
    a.free_state = q.free_state;
    a.free_state_out = q.free_state_out;
    a.pool_bases = q.pool_bases;
    a.block_pointers = q.block_pointers;
    a.token_offsets = q.token_offsets;
    a.slot_map = q.slot_map;
    a.status = q.status;
    a.rows = static_cast<int4*>(q.workspace);
    a.block_bytes = q.block_bytes;
    a.batch = q.batch;
    a.max_blocks = q.max_blocks_per_seq;
    a.num_blocks = q.num_blocks;
    a.num_pools = q.num_pools;
    a.num_tokens = q.num_tokens;
    a.tpb = q.tokens_per_block;
    // the pools are dealt over enough workgroups to fill the chip (a table entry is read once per group)
    a.wgs_per_row = (q.max_blocks_per_seq + 511) / 512;
    const int64_t per_pool = (int64_t) a.wgs_per_row * q.batch;
    const int pool_groups = (int) std::max<int64_t>(1, std::min<int64_t>(q.num_pools, (1024 + per_pool - 1) / per_pool));
    a.pools_per_wg = std::max(1, (q.num_pools + pool_groups - 1) / pool_groups);
    a.planes = (q.num_pools + a.pools_per_wg - 1) / a.pools_per_wg;
    const int64_t grid = per_pool * (a.planes + 1) + ((int64_t) q.num_tokens + 255) / 256;
    MQ_CHECK(grid < (1ll << 24), "block tables: %d requests x %d blocks x %d pools", q.batch, q.max_blocks_per_seq, q.num_pools);
    hipLaunchKernelGGL(table_plan_kernel, dim3(1), dim3(std::min(PLAN_THREADS, (q.batch + 63) / 64 * 64)), 0, stream, a);
    MQ_HIP(hipGetLastError());
    // a table row's pointers two at a time where every row starts on 16 bytes (256 requests of 512 blocks in 64 pools: 26.1 us a
    // call, one at a time 30.8)
    if (q.max_blocks_per_seq % 2 == 0 && (reinterpret_cast<uintptr_t>(q.block_pointers) & 15) == 0)
        hipLaunchKernelGGL(table_fill_kernel<true>, dim3((unsigned) grid), dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL(table_fill_kernel<false>, dim3((unsigned) grid), dim3(256), 0, stream, a);
    MQ_HIP(hipGetLastError());
}

void draft_tree_accept(const mi355q_draft_tree_accept_params& q, hipStream_t stream)
{
    MQ_CHECK(q.batch >= 0 && q.batch <= (1 << 24) && q.num_tokens >= 0 && q.max_path > 0, "batch %d, num_tokens %d, max_path %d", q.batch, q.num_tokens, q.max_path);
    if (q.batch == 0)
        return;
    MQ_CHECK(q.draft_offsets && q.accept_path && q.accept_counts && q.accepted_tokens, "null tensor");
    MQ_CHECK(q.num_tokens == 0 || (q.draft_tokens && q.parents && q.target_tokens), "null tensor");
    hipLaunchKernelGGL(tree_accept_kernel, dim3((q.batch + 3) / 4), dim3(256), 0, stream, q.draft_tokens, q.parents, q.target_tokens,
        q.draft_offsets, q.accept_path, q.accept_counts, q.accepted_tokens, q.batch, q.num_tokens, q.max_path);
    MQ_HIP(hipGetLastError());
}

void kv_commit_path(const mi355q_kv_commit_path_params& q, hipStream_t stream)
{
    MQ_CHECK(q.batch >= 0 && q.batch < (1 << 24) && q.num_pools > 0 && q.num_pools <= 65535 && q.max_path > 0, "batch %d, num_pools %d, max_path %d", q.batch,
        q.num_pools, q.max_path);
    MQ_CHECK(q.max_blocks_per_seq > 0 && q.num_kv_heads > 0, "max_blocks_per_seq %d, num_kv_heads %d", q.max_blocks_per_seq, q.num_kv_heads);
    MQ_CHECK(q.kv_type == MI355Q_HALF || q.kv_type == MI355Q_BF16 || q.kv_type == MI355Q_INT8 || q.kv_type == MI355Q_FP8, "kv cache type %d",
        q.kv_type);
    MQ_CHECK(q.head_size > 0 && q.head_size <= 4096 && q.head_size % 8 == 0, "head_size %d (multiples of 8)", q.head_size);
    const int tpb_log2 = log2_exact(q.tokens_per_block, "tokens_per_block");
    if (q.batch == 0)
        return;
    MQ_CHECK(q.block_pointers && q.past_lengths && q.accept_path && q.accept_counts && q.new_lengths, "null tensor");
    const size_t rows = (size_t) q.batch * sizeof(int32_t);
    // every pool's workgroups read the lengths that pool 0's replace
    MQ_CHECK(!overlap(q.new_lengths, rows, q.past_lengths, rows) && !overlap(q.new_lengths, rows, q.accept_counts, rows)
            && !overlap(q.new_lengths, rows, q.accept_path, rows * q.max_path),
        "new_lengths overlaps an input");
    const int row_bytes = q.head_size * (int) dtype_size(q.kv_type);
    const dim3 g(q.batch, q.num_pools);
    // 16 bytes a lane; 8 where a row is not whole in 16s (the 8-bit caches of head sizes that are odd multiples of 8)
    if (row_bytes % 16 == 0)
        hipLaunchKernelGGL(commit_path_kernel<commit_vec16>, g, dim3(256), 0, stream, q.block_pointers, q.past_lengths, q.accept_path,
            q.accept_counts, q.new_lengths, q.batch, q.max_blocks_per_seq, tpb_log2, q.num_kv_heads, row_bytes, q.max_path);
    else
        hipLaunchKernelGGL(commit_path_kernel<commit_vec8>, g, dim3(256), 0, stream, q.block_pointers, q.past_lengths, q.accept_path,
            q.accept_counts, q.new_lengths, q.batch, q.max_blocks_per_seq, tpb_log2, q.num_kv_heads, row_bytes, q.max_path);
    MQ_HIP(hipGetLastError());
}

} // namespace mi355q
