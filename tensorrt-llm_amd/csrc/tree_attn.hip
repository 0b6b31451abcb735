// tree_attn.hip -- attention of a tree of drafted tokens over the paged cache: the generation step of speculative decoding,
// where the model scores n candidate tokens (nodes) of a sequence at once.
//
// Node i of sequence b is row draft_offsets[b] + i of qkv, sits at position past + position_offsets[row] and owns the cache
// slot past + i.  For every query head
//     out[i] = sum_t softmax_t(q_i . k_t / (sqrt(Dh) q_scaling)) v_t   over t < past and the nodes t = past + j of i's mask,
// and 0 where nothing is visible.  Three launches:
//   1. tree_prepare_kernel: bias and rotation of q, k, v; K / V of every node rounded to the cache's type and stored
//      in its slot; q, times the score scale, to the workspace.  One workgroup per sequence checks its lengths and blocks.
//   2. tree_attn_kernel: flash attention of the nodes over the cache (K / V of the nodes come from the cache too, so a
//      later step over the accepted tokens sees the values that were scored).
//   3. tree_combine_kernel, where the keys of a sequence were split over workgroups: joins the partial states.
#include "attn_mfma.h"
#include "decode_common.h"
#include <type_traits>

namespace mi355q
{
namespace
{

constexpr int TREE_KT = 64;         // keys per tile
constexpr int TREE_THREADS = 256;   // 4 waves
constexpr int TREE_MAX_SPLITS = 128; // parts of a (sequence, kv head): what the combine kernel reads
constexpr int TREE_MAX_DRAFT = 1024;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float TREE_NO_MAX = -FLT_MAX; // the maximum of a state without keys: no finite score lies below it

// The type the products run in: the activation type; fp16 for an 8-bit cache, whose codes it holds exactly (int8 and e4m3 have
// at most 8 significant bits) and in which q and P keep 3 bits more than in bf16.
template <typename T, int KVT>
struct TreeCompute
{
    typedef T type;
};
template <>
struct TreeCompute<bf16_t, 1>
{
    typedef f16_t type;
};
template <>
struct TreeCompute<bf16_t, 2>
{
    typedef f16_t type;
};
// q in two parts (its rounding to the compute type and what that left over): the rotated query would otherwise be the
// largest error beside the result's own rounding.  A bf16 result over fp16 products does not need it.
template <typename T, int KVT>
constexpr bool TREE_Q2 = KVT == 0 || !T16<T>::is_bf16;

struct TreeArgs
{
    const uint16_t* qkv;
    const uint16_t* qkv_bias;
    uint16_t* out;
    const int32_t* past_lengths;
    const int32_t* draft_offsets;
    const int32_t* position_offsets; // or null: the node's index
    const uint32_t* tree_mask;
    const int64_t* block_ptrs;
    const float* kv_scale_orig_quant;
    const float* kv_scale_quant_orig;
    uint16_t* q_ws;      // [tokens][Hq][1 or 2 parts][DP]: rotated, times the score scale (and the K dequantisation) and log2(e)
    int4* order;         // [batch + 1], sequences in the items' order: items before, nodes, first row, history; [batch].x: all items
    int4* split;         // [batch], in the same order: parts of each (sequence, kv head) pair, records before, sequence
    int32_t* seq_ok;     // [batch]: the sequence's blocks are all there
    int4* join;          // [pairs_bound][2]: the pairs of several parts: first row, nodes, kv head, parts (0: none) | record, sequence
    float* part_acc;     // partial states: [record][m-tile][row][DP]
    float2* part_ml;     // their (running maximum in the log2 domain, sum)
    uint8_t* q_shift;    // [tokens][Hq], where the products run in fp16: the query lies in q_ws times 2^-shift
    int64_t qkv_stride;
    int batch, num_heads, num_kv_heads, group, hs;
    int num_tokens, max_draft, max_past, mask_words;
    int max_blocks, tpb_log2;
    int mtiles, rows_per_wg, target_items, part_tiles, items_bound, pairs_bound;
    int whole; // every (sequence, kv head) is one item: nothing is joined
    int pos_type, rot_dim, rot_scale_type, rot_max_pos;
    double rot_log2_base, rot_scale;
    float score_scale;
};

// The sequence's rows, from device memory: false when the lengths do not fit what the host was told, so that nothing is
// read or written outside the tensors (such a sequence is skipped).
__device__ __forceinline__ bool tree_seq(const TreeArgs& p, int b, int& off, int& n, int& past)
{
    off = p.draft_offsets[b];
    n = p.draft_offsets[b + 1] - off;
    past = p.past_lengths[b];
    const int64_t end = (int64_t) off + n, keys = (int64_t) past + n;
    return off >= 0 && n > 0 && n <= p.max_draft && end <= p.num_tokens && past >= 0 && past <= p.max_past
        && keys <= ((int64_t) p.max_blocks << p.tpb_log2);
}

// The items of the attention kernel, by one workgroup: a (sequence, kv head) pair is cut into parts of about equally many tiles, so
// many that about target_items come out (part_tiles: the least a part should have; -1 times the most if the caller says how many).
// Sequences with long parts come first (up to 256 sequences), so that what is left for the end is short: 16 sequences of 680 .. 4100
// tokens, 64 nodes, 64 / 8 heads 161 -> 132 us; 64 of 1000 .. 6000, 4 nodes, 32 / 8 heads, fp8 127 -> 113; equal lengths +0.3 us.
__device__ __forceinline__ void tree_plan_items(const TreeArgs& p)
{
    constexpr int WAVES = TREE_THREADS / 64;
    __shared__ int wave_sum[3][WAVES];
    __shared__ int part_len[TREE_THREADS], sorted_parts[TREE_THREADS];
    __shared__ int4 sorted[TREE_THREADS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, H = p.num_kv_heads;
    auto tiles = [&](int b, int& off, int& n, int& past)
    { return b < p.batch && tree_seq(p, b, off, n, past) ? (past + n + TREE_KT - 1) / TREE_KT : 0; };
    int target = p.whole ? INT32_MAX : -p.part_tiles;
    if (!p.whole && p.part_tiles > 0)
    {
        int all = 0, off, n, past;
        for (int b = threadIdx.x; b < p.batch; b += TREE_THREADS)
            all += tiles(b, off, n, past);
#pragma unroll
        for (int o = 32; o; o >>= 1)
            all += __shfl_xor(all, o);
        if (lane == 0)
            wave_sum[0][wave] = all;
        __syncthreads();
        all = 0;
        for (int w = 0; w < WAVES; ++w)
            all += wave_sum[0][w];
        target = max((all * H + p.target_items - 1) / p.target_items, p.part_tiles);
        __syncthreads();
    }
    int carry[3] = {0, 0, 0}; // items, records, pairs of several parts
    for (int b0 = 0; b0 < p.batch; b0 += TREE_THREADS)
    {
        const int b = b0 + threadIdx.x;
        int off = 0, n = 0, past = 0;
        const int nt = tiles(b, off, n, past);
        int parts = 0;
        if (nt > 0)
            parts = p.whole ? 1 : (p.part_tiles < 0 ? (nt - 1) / target + 1 : max((2 * nt + target) / (2 * target), 1));
        int seq = b;
        if (p.batch > 1 && p.batch <= TREE_THREADS)
        {
            const int len = nt > 0 ? (nt - 1) / parts + 1 : 0;
            part_len[threadIdx.x] = len;
            __syncthreads();
            int rank = b;
            if (b < p.batch)
            {
                rank = 0;
                for (int j = 0; j < p.batch; ++j)
                    rank += part_len[j] > len || (part_len[j] == len && j < b);
            }
            sorted[rank] = make_int4(n, off, past, b);
            sorted_parts[rank] = parts;
            __syncthreads();
            const int4 x = sorted[threadIdx.x];
            n = x.x, off = x.y, past = x.z, seq = x.w;
            parts = sorted_parts[threadIdx.x];
        }
        const int mine[3] = {parts * H, parts > 1 ? parts * H : 0, parts > 1 ? H : 0};
        int x[3] = {mine[0], mine[1], mine[2]};
#pragma unroll
        for (int o = 1; o < 64; o <<= 1)
#pragma unroll
            for (int i = 0; i < 3; ++i)
            {
                const int y = __shfl_up(x[i], o);
                x[i] += lane >= o ? y : 0;
            }
        if (lane == 63)
#pragma unroll
            for (int i = 0; i < 3; ++i)
                wave_sum[i][wave] = x[i];
        __syncthreads();
        int before[3];
#pragma unroll
        for (int i = 0; i < 3; ++i)
        {
            before[i] = carry[i] + x[i] - mine[i];
            for (int w = 0; w < WAVES; ++w)
            {
                before[i] += w < wave ? wave_sum[i][w] : 0;
                carry[i] += wave_sum[i][w];
            }
        }
        if (b < p.batch)
        {
            p.order[b] = make_int4(before[0], parts ? n : 0, off, past);
            p.split[b] = make_int4(parts, before[1], seq, 0);
            for (int h = 0; h < (parts > 1 ? H : 0); ++h)
            {
                p.join[2 * (before[2] + h)] = make_int4(off, n, h, parts);
                p.join[2 * (before[2] + h) + 1] = make_int4(before[1] + h * parts, seq, 0, 0);
            }
        }
        __syncthreads();
    }
    if (threadIdx.x == 0)
        p.order[p.batch] = make_int4(carry[0], 0, 0, 0);
    for (int i = carry[2] + threadIdx.x; i < p.pairs_bound; i += TREE_THREADS)
        p.join[2 * i] = make_int4(0, 0, 0, 0);
}

// 8 elements from d0 on of one head of a qkv row, bias added, rotated: in fp32 or in 64 bits (R).  angle(j, c, s) gives cosine
// and sine of pair j.
template <typename T, typename R, typename Angle>
__device__ __forceinline__ void tree_chunk8(
    const TreeArgs& p, const uint16_t* src, int vec, int d0, int half, bool rope, R (&y)[8], Angle&& angle)
{
    const int at = vec * p.hs;
    auto elements = [&](int d, R (&x)[8])
    {
        const uint4 r = *reinterpret_cast<const uint4*>(src + at + d);
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int e = 0; e < 8; ++e)
            x[e] = (e & 1) ? T16<T>::hi(w[e >> 1]) : T16<T>::lo(w[e >> 1]);
        if (p.qkv_bias)
        {
            const uint4 rb = *reinterpret_cast<const uint4*>(p.qkv_bias + at + d);
            const uint32_t wb[4] = {rb.x, rb.y, rb.z, rb.w};
#pragma unroll
            for (int e = 0; e < 8; ++e)
                x[e] += (e & 1) ? T16<T>::hi(wb[e >> 1]) : T16<T>::lo(wb[e >> 1]);
        }
    };
    elements(d0, y);
    if (!rope || d0 >= p.rot_dim)
        return;
    R c, s;
    if (p.pos_type == 1) // GPT-J pairs (2 j, 2 j + 1)
    {
#pragma unroll
        for (int e = 0; e < 8; e += 2)
            if (d0 + e < p.rot_dim)
            {
                angle((d0 + e) >> 1, c, s);
                const R a = y[e], b = y[e + 1];
                y[e] = a * c - b * s;
                y[e + 1] = b * c + a * s;
            }
    }
    else if (half % 8 == 0) // NeoX pairs (j, j + rot_dim / 2): the partners are a chunk of their own
    {
        const bool first = d0 < half;
        R other[8];
        elements(first ? d0 + half : d0 - half, other);
#pragma unroll
        for (int e = 0; e < 8; ++e)
        {
            angle(d0 + e - (first ? 0 : half), c, s);
            y[e] = y[e] * c + (first ? -other[e] : other[e]) * s;
        }
    }
    else
    {
#pragma unroll
        for (int e = 0; e < 8; ++e)
        {
            const int d = d0 + e;
            if (d < p.rot_dim)
            {
                const bool first = d < half;
                const int o = at + (first ? d + half : d - half);
                R other = T16<T>::to_float(src[o]);
                if (p.qkv_bias)
                    other += T16<T>::to_float(p.qkv_bias[o]);
                angle(first ? d : d - half, c, s);
                y[e] = y[e] * c + (first ? -other : other) * s;
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------- 1. prepare
// grid (max_draft + 2, batch, parts of the heads).  Angles, and rotation and quantisation of K / V, run in 64 bits: the angle of a
// far position has few correct digits left in fp32 (position 2^17: error 2^-8 rad).  From there K / V go through fp32 to the cache's type,
// as torch's conversion does (int8 codes are rounded in 64 bits): the stored rows equal those of the definition.
// The queries, the larger part, are rotated in fp32.
// Bound by memory: rows in, two parts of q and K / V out, in rows of 256 bytes.  708 tokens of 32 + 64 heads of 128: 14 us for 41 MB;
// 8 tokens: 4.0 us, a launch, three dependent loads and the angles.  (Loading a thread's elements ahead of the angles, values
// as plain copies, and more or fewer workgroups than 2048 all cost 1 to 3 us more.)
template <typename T, int KVT>
__global__ __launch_bounds__(TREE_THREADS) void tree_prepare_kernel(TreeArgs p, int dp)
{
    typedef typename TreeCompute<T, KVT>::type C;
    constexpr int PARTS = TREE_Q2<T, KVT> ? 2 : 1;
    const int b = blockIdx.y, i = blockIdx.x;
    int off, n, past;
    if (i == p.max_draft + 1)
    {
        if (b == 0 && blockIdx.z == 0)
            tree_plan_items(p);
        return;
    }
    const bool ok = tree_seq(p, b, off, n, past);
    const int tpb = 1 << p.tpb_log2;
    const int64_t* kp = p.block_ptrs + (size_t) b * 2 * p.max_blocks;
    if (i == p.max_draft)
    {
        if (blockIdx.z > 0)
            return;
        // every block the sequence's keys live in has to be there (0 = not allocated) and aligned like the loads from it
        bool bad = !ok;
        if (ok)
            for (int j = threadIdx.x; j < (past + n + tpb - 1) >> p.tpb_log2; j += TREE_THREADS)
                bad |= kp[j] == 0 || kp[p.max_blocks + j] == 0 || ((kp[j] | kp[p.max_blocks + j]) & 15) != 0;
        bad = __syncthreads_or(bad);
        if (threadIdx.x == 0)
            p.seq_ok[b] = !bad;
        return;
    }
    if (!ok || i >= n)
        return;
    const int row = off + i, hs = p.hs;
    const int Hq = p.num_heads, Hkv = p.num_kv_heads;
    const bool rope = p.pos_type == 1 || p.pos_type == 2;
    const int half = p.rot_dim >> 1;
    __shared__ double cs_tab[128], sn_tab[128];
    __shared__ float2 q_tab[128]; // the same in fp32, for the queries
    if (rope && (int) threadIdx.x < half)
    {
        const int pos = past + (p.position_offsets ? p.position_offsets[row] : i);
        double log2_base = p.rot_log2_base, scale = p.rot_scale;
        if (p.rot_scale_type == 2) // dynamic NTK: the base grows with the length once that passes the trained one
        {
            if (pos > p.rot_max_pos)
                log2_base += log2(pos * (scale / p.rot_max_pos) - (scale - 1.0)) * p.rot_dim / (p.rot_dim - 2);
            scale = 1.0;
        }
        else if (p.rot_scale_type == 1)
            scale = 1.0 / scale;
        else
            scale = 1.0;
        const double turns = pos * scale * exp2(-log2_base * (2 * (int) threadIdx.x) / p.rot_dim) * 0.15915494309189535;
        double sn, cs;
        sincospi(2.0 * (turns - rint(turns)), &sn, &cs);
        cs_tab[threadIdx.x] = cs;
        sn_tab[threadIdx.x] = sn;
        q_tab[threadIdx.x] = make_float2((float) cs, (float) sn);
    }
    __syncthreads();
    const uint16_t* src = p.qkv + (size_t) row * p.qkv_stride;
    const int cpv = dp / 8, nvec = Hq + 2 * Hkv; // 8-element chunks per head
    const float qscale = p.score_scale * LOG2E * (KVT ? p.kv_scale_quant_orig[0] : 1.f);
    const double kvq = KVT ? (double) p.kv_scale_orig_quant[0] : 1.0;
    const int slot = past + i, blk = slot >> p.tpb_log2, tin = slot & (tpb - 1);
    char* const kdst = reinterpret_cast<char*>(kp[blk]);
    char* const vdst = reinterpret_cast<char*>(kp[p.max_blocks + blk]);
    for (int it = blockIdx.z * TREE_THREADS + threadIdx.x; it < nvec * cpv; it += gridDim.z * TREE_THREADS)
    {
        const int vec = it / cpv, d0 = 8 * (it % cpv);
        uint4* const qdst = reinterpret_cast<uint4*>(p.q_ws + ((size_t) row * Hq + vec) * PARTS * dp + d0);
        if (vec >= Hq && d0 >= hs)
            continue;
        if (vec < Hq)
        {
            // q carries the score scale, the K dequantisation and log2(e): the matrix product then IS the exponent
            float z[8] = {}, hi[8], lo[8]; // (zeros: the padding of the workspace rows)
            if (d0 < hs)
            {
                float y[8];
                tree_chunk8<T>(p, src, vec, d0, half, rope, y, [&](int j, float& c, float& s) { c = q_tab[j].x, s = q_tab[j].y; });
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    z[e] = y[e] * qscale;
            }
            if constexpr (!T16<C>::is_bf16)
            {
                // a head whose largest element (infinities apart) fp16 does not hold goes down by a power of 2, which the scores get
                // back in fp32.  The lanes of a head are neighbours in one wave
                float top = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    top = fmaxf(top, fabsf(z[e]) < HUGE_VALF ? fabsf(z[e]) : 0.f);
                int shift = 0;
                if (__any(top > 65504.f))
                {
                    for (int o = 1; o < cpv; o <<= 1)
                        top = fmaxf(top, __shfl_xor(top, o));
                    shift = top > 65504.f ? ilogbf(top) - 14 : 0;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        z[e] = ldexpf(z[e], -shift);
                }
                if (d0 == 0)
                    p.q_shift[(size_t) row * Hq + vec] = shift;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                hi[e] = T16<C>::to_float(T16<C>::from_float(z[e]));
                lo[e] = fabsf(hi[e]) < HUGE_VALF ? z[e] - hi[e] : 0.f;
            }
            *qdst = make_uint4(pack2<C>(hi[0], hi[1]), pack2<C>(hi[2], hi[3]), pack2<C>(hi[4], hi[5]), pack2<C>(hi[6], hi[7]));
            if constexpr (PARTS == 2)
                qdst[dp / 8] = make_uint4(pack2<C>(lo[0], lo[1]), pack2<C>(lo[2], lo[3]), pack2<C>(lo[4], lo[5]), pack2<C>(lo[6], lo[7]));
            continue;
        }
        double y[8];
        tree_chunk8<T>(p, src, vec, d0, half, rope && vec < Hq + Hkv, y, [&](int j, double& c, double& s) { c = cs_tab[j], s = sn_tab[j]; });
        const int kv = (vec - Hq) / Hkv, hk = (vec - Hq) % Hkv;
        char* const base = kv ? vdst : kdst;
        if (!base || (reinterpret_cast<uintptr_t>(base) & 15))
            continue;
        const size_t e0 = ((size_t) hk * tpb + tin) * hs + d0;
        if constexpr (KVT == 0)
        {
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                o[e] = pack2<T>((float) y[2 * e], (float) y[2 * e + 1]);
            *reinterpret_cast<uint4*>(base + 2 * e0) = make_uint4(o[0], o[1], o[2], o[3]);
        }
        else
        {
            uint32_t o[2] = {0, 0};
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                const double z = y[e] * kvq;
                const uint32_t c = KVT == 1 ? float_to_int8_sat((float) rint(z)) : float_to_fp8((float) z);
                o[e >> 2] |= c << (8 * (e & 3));
            }
            *reinterpret_cast<uint2*>(base + e0) = make_uint2(o[0], o[1]);
        }
    }
}

// ---------------------------------------------------------------------------------------------- 2. attention
template <typename T>
__device__ __forceinline__ cf32x4_t tree_mfma16(const uint2& a, const uint2& b, cf32x4_t c);
template <>
__device__ __forceinline__ cf32x4_t tree_mfma16<bf16_t>(const uint2& a, const uint2& b, cf32x4_t c)
{
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(
        __builtin_bit_cast(cs16x4_t, a), __builtin_bit_cast(cs16x4_t, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ cf32x4_t tree_mfma16<f16_t>(const uint2& a, const uint2& b, cf32x4_t c)
{
    typedef __attribute__((ext_vector_type(4))) _Float16 f16x4_t;
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4_t, a), __builtin_bit_cast(f16x4_t, b), c, 0, 0, 0);
}

// 8 cache bytes -> 8 fp16 values (exact)
template <int KVT>
__device__ __forceinline__ uint4 tree_kv8_to_f16(uint32_t w0, uint32_t w1)
{
    uint4 r;
    if constexpr (KVT == 2)
    {
        r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.f, false));
        r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.f, true));
        r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.f, false));
        r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.f, true));
    }
    else
    {
        r.x = pack2<f16_t>(kv8_to_float<1>(w0, 0), kv8_to_float<1>(w0, 1));
        r.y = pack2<f16_t>(kv8_to_float<1>(w0, 2), kv8_to_float<1>(w0, 3));
        r.z = pack2<f16_t>(kv8_to_float<1>(w1, 0), kv8_to_float<1>(w1, 1));
        r.w = pack2<f16_t>(kv8_to_float<1>(w1, 2), kv8_to_float<1>(w1, 3));
    }
    return r;
}

// 16 bytes of the LDS from a byte address
__device__ __forceinline__ uint4 tree_lds16(uint32_t address)
{
    typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_t;
    const u32x4_t v = *(const __attribute__((address_space(3))) u32x4_t*) (uintptr_t) address;
    return make_uint4(v.x, v.y, v.z, v.w);
}

// 16 bytes from an address that was an integer in a table: a global load (a plain cast would make it a flat one)
__device__ __forceinline__ uint4 tree_load16(int64_t address)
{
    typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_t;
    const u32x4_t v = *(const __attribute__((address_space(1))) u32x4_t*) address;
    return make_uint4(v.x, v.y, v.z, v.w);
}

// the LDS-DMA of ctx_dma16 with a wave-uniform base and a 32-bit lane offset
__device__ __forceinline__ void tree_dma16(int64_t base, uint32_t offset, uint32_t lds_off)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(lds_off) : "memory", "m0");
}

// does a dword of two T values hold an infinity or NaN
template <typename T>
__device__ __forceinline__ bool tree_nonfinite2(uint32_t w)
{
    constexpr uint32_t EXP = T16<T>::is_bf16 ? 0x7f80u : 0x7c00u;
    return (w & EXP) == EXP || ((w >> 16) & EXP) == EXP;
}

// 64 bits of a mask row from bit `s0` on; bits below 0 (keys of the history) read as 1, past the row as 0
__device__ __forceinline__ uint64_t tree_mask64(const uint32_t* row, int words, int n, int s0)
{
    uint64_t v = 0;
    const int w0 = s0 >> 5, sh = s0 & 31; // arithmetic shift: floor
    uint32_t w[3];
#pragma unroll
    for (int i = 0; i < 3; ++i)
    {
        const int j = w0 + i;
        w[i] = (j >= 0 && j < words) ? row[j] : 0u;
    }
    v = ((uint64_t) w[1] << 32 | w[0]) >> sh;
    if (sh)
        v |= (uint64_t) w[2] << (64 - sh);
    if (s0 < 0)
        v |= (1ull << -s0) - 1; // (s0 > -64)
    const int live = n - s0; // keys of the window that exist
    return live >= 64 ? v : (live <= 0 ? 0ull : v & ((1ull << live) - 1));
}

// grid: 1-D, ((item / 8) * mtiles + m) * 8 + item % 8: workgroups are dealt to the 8 XCDs round-robin, so the m-tiles of an item, which
// walk the same keys, run on one XCD and read them from HBM once.
// An item is a (sequence, kv head) pair or a part of its key tiles.  Whole pairs write their output; parts leave their state
// for the combine kernel.
// A workgroup = RW * QT * 16 query rows (row r = node r / G, head r % G of the kv head's G query heads).  Its 4 waves are RW row
// groups x KW key groups: with few rows the waves share the keys of a tile instead of idling, and merge their states at
// the end.
// S^T = K . Q^T (16x16x32): a lane holds one query column's scores of 4 consecutive keys, and the same registers, rounded
// to the compute type, are the B operand of O^T += V^T . P^T.
// Softmax in the log2 domain with the running maximum m as the C operand of the first product: what comes out is already
// s - m, and as long as no column grows past m + 8 (p <= 256: harmless in bf16 and in the fp32 sums) nothing is rescaled.
// fp16 has few numbers below 1 and many above: there m lies 10 below the largest score, p goes up to 2^15, and the weights keep
// their bits down to 2^-24 of the largest and vanish below 2^-35 (with m at the largest 2^-14 and 2^-25: many keys far behind
// a single one were lost).  It costs nothing: the times of all fp16 and 8-bit cases stayed.
// Whether one does is an integer maximum over the raw bits (negative floats are negative integers).
// Scores that come out NaN: an infinite key element, or products beyond fp32, meet the second part of q, whose sign is either, or
// the zeros that q is padded with.  The row's sum is then NaN, and the whole item runs again with careful scores; what is still
// NaN then is so by the definition.  So does an item with a query that was shifted into the range of fp16.
// Two workgroups live on a CU (64 KiB of LDS: a tile of K and V that is computed, one that arrives), 2 waves a SIMD at 225 to 255
// registers; what one waits for the other covers.  Bound by HBM up to some 32 rows a kv head, then by the matrix instructions,
// of which the second part of q is a third, by the softmax beside them and by the LDS.  Whole calls, bf16, Dh 128, 64 sequences of 2048
// tokens, 32 / 32 heads: 1 node 5.7 TB/s, 16 nodes 5.3, 64 nodes 4.8 (a copy reaches 5.05); 16 x 4096 tokens, 64 nodes, 64 / 8 heads:
// 199 us = 0.70 PFLOP/s of the formula's and 1.05 of products issued (a large matrix product 1.23); one sequence of 120001
// tokens, 60 nodes, 64 / 8 heads: 308 to 317 us, matrix pipes busy 53 %, no LDS conflicts.  Four tiles in flight with one workgroup a CU
// took 127 us where this took 93, 8 waves of 256 rows 275 for 217.
template <typename T, int KVT, int DP, int RW, int KW, int QT>
__global__ __launch_bounds__(TREE_THREADS) __attribute__((amdgpu_waves_per_eu(DP > 128 ? 1 : 2))) void tree_attn_kernel(TreeArgs p)
{
    static_assert(RW * KW == 4, "4 waves");
    typedef typename TreeCompute<T, KVT>::type C;
    constexpr int PARTS = TREE_Q2<T, KVT> ? 2 : 1;
    constexpr int M = RW * QT * 16;
    constexpr int KS = DP / 32, DT = DP / 16;
    constexpr int ROWB = DP * 2, CH = ROWB / 16;
    constexpr int TILE_BYTES = TREE_KT * ROWB, STAGE_BYTES = 2 * TILE_BYTES;
    constexpr int XW = 4 / KW;                      // 16-key subtiles per wave
    constexpr int X2 = XW < 2 ? XW : 2;             // subtiles per compute step: 32 keys, or 16 with four key groups
    constexpr float LEAD = T16<C>::is_bf16 ? 0.f : 10.f;                       // m below the largest score when it is set
    constexpr int GROWTH = __builtin_bit_cast(int, T16<C>::is_bf16 ? 8.f : 15.f); // s - m from which on the column is rescaled
    // fragments read from the LDS ahead of their products, as many as the registers hold (8-bit caches hold a tile in them too)
    constexpr bool TIGHT = KVT && PARTS == 2 && QT == 2 && DP >= 128;
    constexpr int KBATCH = TIGHT && X2 == 2 ? 2 : KS, VBATCH = TIGHT && X2 == 2 ? 4 : (DT < 8 ? DT : 8);
    constexpr int WROWS = TREE_KT / 4;              // a wave loads 16 consecutive keys of a tile
    constexpr int RPD = 1024 / ROWB, DPW = WROWS / RPD; // 16-bit caches: rows per DMA instruction, DMAs per wave
    constexpr int CH8 = DP / 16, RPL = 64 / CH8, LPT = WROWS / RPL; // 8-bit caches: rows per 16-byte load, loads per thread
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * STAGE_BYTES]; // a tile that is computed, a tile that arrives
    __shared__ uint32_t nonfinite[TREE_MAX_DRAFT / 32]; // nodes whose V row has an infinity or NaN
    __shared__ int redo;                                // a row's sum is NaN, or its query shifted

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rw = wave % RW, kw = wave / RW;
    const int lr = lane & 15, lq = lane >> 4;
    const int mt = (blockIdx.x >> 3) % p.mtiles;
    const int item = (blockIdx.x >> 3) / p.mtiles * 8 + (blockIdx.x & 7);
    if (item >= p.items_bound)
        return;
    const int G = p.group, hs = p.hs, tpb_mask = (1 << p.tpb_log2) - 1;
    const int row_bytes = hs * (KVT ? 1 : 2); // of a head in the cache

    // swizzle of the 16-byte chunk index by the row, K and V alike.  The banks see a 16-byte read of 64 lanes in groups of rows
    // 0-3, 12-15 at one chunk with rows 4-11 at its neighbour (K fragments: row = lane & 15), and a transposing read in groups of
    // 4 rows x 2 chunks (V): both fall on all banks once.  The tile writes of the 8-bit caches, every other chunk of two neighbouring
    // rows, do not: a quarter of that kernel's LDS cycles are conflicts.  It depends on the row modulo 16 only.
    auto sw = [](int row)
    {
        const int x = (row >> 2) & 3;
        return CH >= 16 ? (row & 3) << 2 | ((x ^ x >> 1) & 1) << 1 | (x >> 1 ^ (row & 1)) : ((row >> 1) & 3) << 1;
    };

    // ---- the item's sequence.  64 lanes look at the items before 64 sequences (or before every len / 64th of more)
    int b0 = 0;
    if (p.whole)
        b0 = item / p.num_kv_heads & ~63;
    else
        for (int len = p.batch; len > 64;)
        {
            const int step = (len + 63) / 64;
            const int at = b0 + (lane + 1) * step;
            b0 += step * __builtin_popcountll(__ballot(at < p.batch && p.order[min(at, p.batch)].x <= item));
            len = step;
        }
    const int4 info = p.order[min(b0 + lane, p.batch)];
    const int info_next = p.order[min(b0 + lane + 1, p.batch)].x;
    const int4 info_split = p.split[min(b0 + lane, p.batch - 1)];
    const int at = __builtin_amdgcn_readfirstlane(
        p.whole ? item / p.num_kv_heads - b0 : __builtin_popcountll(__ballot(b0 + lane < p.batch && info_next <= item)));
    if (b0 + at >= p.batch) // behind the last item
        return;
    const int b = __builtin_amdgcn_readlane(info_split.z, at), n = __builtin_amdgcn_readlane(info.y, at);
    if (mt * M >= n * G) // an empty sequence, or no rows for this m-tile
        return;
    const int off = __builtin_amdgcn_readlane(info.z, at), past = __builtin_amdgcn_readlane(info.w, at), total = past + n;
    const int nt = (total + TREE_KT - 1) / TREE_KT, parts = __builtin_amdgcn_readlane(info_split.x, at);
    const int in_seq = p.whole ? item % p.num_kv_heads : item - __builtin_amdgcn_readlane(info.x, at);
    const int head_kv = in_seq / parts, part_no = in_seq % parts;
    const int tile_lo = nt / parts * part_no + min(part_no, nt % parts), tile_hi = tile_lo + nt / parts + (part_no < nt % parts);
    const int64_t* const kp = p.block_ptrs + (size_t) b * 2 * p.max_blocks;
    const int64_t* const vp = kp + p.max_blocks;
    const bool long_tree = n > 64;

    // ---- LDS and cache offsets
    const uint32_t lds_base = __builtin_amdgcn_readfirstlane((uint32_t) (uintptr_t) (ctx_lds_void_t*) lds);
    const int last_chunk = row_bytes / 16 - 1; // heads narrower than DP: the padding re-reads the last chunk (q is 0 there)
    constexpr int LOADS = KVT ? LPT : DPW;
    uint32_t lane_off[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
    {
        const int r = i * (KVT ? RPL : RPD) + lane / (KVT ? CH8 : CH); // row of the wave's 16
        const int ch = lane % (KVT ? CH8 : CH);
        lane_off[i] = r * row_bytes + 16 * min(KVT ? ch : ch ^ sw(r), last_chunk);
    }
    const int rq = lr >> 2, rp = lr & 3;
    const int kb0 = kw * 16 * XW; // this wave's first key of a tile
    // LDS addresses of a lane's fragments in stage 0: K row lr, chunk lq (+ 4 ks by XOR); V row 4 lq + rq, column 4 rp (+ 16 dt by XOR)
    const uint32_t k_addr = lds_base + ROWB * (kb0 + lr) + 16 * (lq ^ sw(lr));
    const uint32_t v_addr = lds_base + TILE_BYTES + ROWB * (kb0 + 4 * lq + rq) + 16 * ((rp >> 1) ^ sw(4 * lq + rq)) + 8 * (rp & 1);
    typedef const __attribute__((address_space(4))) int64_t* scalar_ptr;

    // ---- tile loads.  A wave loads 16 consecutive keys, which lie in one block (tokens_per_block >= 16): the block's address
    // is a scalar load, issued a tile ahead, and a lane adds a fixed 32-bit offset.  16-bit caches: LDS-DMA, instruction d of
    // a tile fills LDS bytes [1024 d, +1024), the swizzle applied on the source address.  8-bit caches: through registers,
    // converted on the way into the LDS.  Keys past the sequence are whatever its last block holds there.
    int64_t kbase = 0, vbase = 0; // where the wave's 16 keys of the tile to be loaded next begin
    auto find_tile = [&](int i)
    {
        const int t0 = i * TREE_KT + wave * WROWS;
        const int blk = __builtin_amdgcn_readfirstlane(min(t0, total - 1) >> p.tpb_log2);
        const int64_t in_block = (((int64_t) head_kv << p.tpb_log2) + (t0 & tpb_mask)) * row_bytes;
        kbase = ((scalar_ptr) kp)[blk] + in_block;
        vbase = ((scalar_ptr) vp)[blk] + in_block;
    };
    uint4 kreg[KVT ? LPT : 1], vreg[KVT ? LPT : 1];
    auto load_tile = [&](uint32_t stage)
    {
#pragma unroll
        for (int d = 0; d < LOADS; ++d)
        {
            if constexpr (KVT == 0)
            {
                const uint32_t dst = lds_base + stage + (wave * DPW + d) * 1024;
                tree_dma16(kbase, lane_off[d], dst);
                tree_dma16(vbase, lane_off[d], dst + TILE_BYTES);
            }
            else
            {
                kreg[d] = tree_load16(kbase + lane_off[d]);
                vreg[d] = tree_load16(vbase + lane_off[d]);
            }
        }
    };
    auto store_tile = [&](uint32_t stage) // 8-bit caches
    {
        if constexpr (KVT != 0)
        {
#pragma unroll
            for (int d = 0; d < LPT; ++d)
            {
                const int r = d * RPL + lane / CH8, ch = 2 * (lane % CH8);
                uint8_t* kt = lds + stage + ROWB * (wave * WROWS + r);
                uint8_t* vt = kt + TILE_BYTES;
                *reinterpret_cast<uint4*>(kt + 16 * (ch ^ sw(r))) = tree_kv8_to_f16<KVT>(kreg[d].x, kreg[d].y);
                *reinterpret_cast<uint4*>(kt + 16 * ((ch + 1) ^ sw(r))) = tree_kv8_to_f16<KVT>(kreg[d].z, kreg[d].w);
                *reinterpret_cast<uint4*>(vt + 16 * (ch ^ sw(r))) = tree_kv8_to_f16<KVT>(vreg[d].x, vreg[d].y);
                *reinterpret_cast<uint4*>(vt + 16 * ((ch + 1) ^ sw(r))) = tree_kv8_to_f16<KVT>(vreg[d].z, vreg[d].w);
            }
        }
    };

    // (the barrier of the first tile comes before the first use)
    if (KVT == 0 && tid < TREE_MAX_DRAFT / 32)
        nonfinite[tid] = 0;
    if (tid == 0)
        redo = 0;
    find_tile(tile_lo);
    if (!p.seq_ok[b]) // a block is missing: nothing of it is read
        return;
    load_tile(0);
    find_tile(min(tile_lo + 1, tile_hi - 1));
    // ---- Q^T fragments (B operand): column = row q0 + 16 qt + lr, k = d = 32 ks + 8 lq + j
    const int q0 = mt * M + rw * QT * 16;
    uint4 qf[PARTS][QT][KS];
    uint64_t mask_row[QT]; // the first 64 nodes' bits
    int q_shift[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
    {
        const int r = min(q0 + 16 * qt + lr, n * G - 1); // rows past the last re-read it; never stored
        const uint32_t* mrow = p.tree_mask + (size_t) (off + r / G) * p.mask_words;
        mask_row[qt] = (uint64_t) mrow[p.mask_words > 1 ? 1 : 0] << 32 | mrow[0];
        if (n < 64)
            mask_row[qt] &= (1ull << n) - 1;
        const size_t head = (size_t) (off + r / G) * p.num_heads + head_kv * G + r % G;
        const uint16_t* q = p.q_ws + head * PARTS * DP;
        q_shift[qt] = 0;
        if constexpr (!T16<C>::is_bf16)
            q_shift[qt] = p.q_shift[head];
#pragma unroll
        for (int part = 0; part < PARTS; ++part)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                qf[part][qt][ks] = *reinterpret_cast<const uint4*>(q + part * DP + 32 * ks + 8 * lq);
    }
    // end the compiler's own bookkeeping of these loads here, before the loop's (to it invisible) DMAs
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
        asm volatile("" : "+v"(mask_row[qt]), "+v"(q_shift[qt]));
#pragma unroll
    for (int part = 0; part < PARTS; ++part)
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                asm volatile("" : "+v"(qf[part][qt][ks].x), "+v"(qf[part][qt][ks].y), "+v"(qf[part][qt][ks].z), "+v"(qf[part][qt][ks].w));

    float l_run[QT];
    cf32x4_t minus_m[QT]; // C operand of the scores: minus the running maximum
    bool fresh[QT];       // the column has no maximum yet (minus_m is 0)
    cf32x4_t o[QT][DT];

    // One compute step: X2 subtiles from key `kb` of the tile in `stage` on.  GENERAL: columns may still be fresh, keys hidden.
    bool careful = false;
    auto step = [&](auto general, uint32_t stage, int kb, int t0)
    {
        constexpr bool GENERAL = decltype(general)::value;
        const uint32_t ka = k_addr + stage + kb * ROWB, va = v_addr + stage + kb * ROWB;
        cf32x4_t s[X2][QT];
#pragma unroll
        for (int x = 0; x < X2; ++x)
#pragma unroll
            for (int qt = 0; qt < QT; ++qt)
                s[x][qt] = minus_m[qt];
        if (GENERAL && careful) // uniform
        {
            // the products of the two parts of q apart, the padding of the keys as zeros; the second part counts only where both are
            // finite, so that an infinite score keeps the sign that the first part gives it; a shifted query's scores shifted back
#pragma unroll 1
            for (int x = 0; x < X2; ++x)
#pragma unroll
                for (int qt = 0; qt < QT; ++qt)
                {
                    cf32x4_t hi = {0.f, 0.f, 0.f, 0.f}, lo = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
                    {
                        uint4 kf = tree_lds16((ka ^ (64 * ks)) + 16 * x * ROWB);
                        if (32 * ks + 8 * lq >= hs)
                            kf = make_uint4(0, 0, 0, 0);
                        hi = ctx_mfma<C>(kf, qf[0][qt][ks], hi);
                        if constexpr (PARTS == 2)
                            lo = ctx_mfma<C>(kf, qf[PARTS - 1][qt][ks], lo);
                    }
#pragma unroll
                    for (int rr = 0; rr < 4; ++rr)
                    {
                        const float z = fabsf(hi[rr]) < HUGE_VALF && fabsf(lo[rr]) < HUGE_VALF ? hi[rr] + lo[rr] : hi[rr];
#pragma unroll
                        for (int y = 0; y < X2; ++y)
                            s[y][qt][rr] = y == x ? ldexpf(z, q_shift[qt]) + minus_m[qt][rr] : s[y][qt][rr];
                    }
                }
        }
        else
#pragma unroll
            for (int ks0 = 0; ks0 < KS; ks0 += KBATCH)
            {
                uint4 kf[KBATCH][X2];
#pragma unroll
                for (int ks = 0; ks < KBATCH; ++ks)
#pragma unroll
                    for (int x = 0; x < X2; ++x)
                        kf[ks][x] = tree_lds16((ka ^ (64 * (ks0 + ks))) + 16 * x * ROWB);
#pragma unroll
                for (int ks = 0; ks < KBATCH; ++ks)
#pragma unroll
                    for (int part = PARTS - 1; part >= 0; --part)
#pragma unroll
                        for (int x = 0; x < X2; ++x) // consecutive products go to different accumulators
#pragma unroll
                            for (int qt = 0; qt < QT; ++qt)
                                s[x][qt] = ctx_mfma<C>(kf[ks][x], qf[part][qt][ks0 + ks], s[x][qt]);
            }
        // the first V fragments are read while the softmax runs
        uint2 vf[VBATCH][X2];
        auto read_v = [&](int d0)
        {
#pragma unroll
            for (int dt = 0; dt < VBATCH; ++dt)
#pragma unroll
                for (int x = 0; x < X2; ++x)
                    vf[dt][x] = __builtin_bit_cast(uint2,
                        __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_cs16x4_t*) (uintptr_t) ((va ^ (32 * (d0 + dt))) + 16 * x * ROWB)));
        };
        read_v(0);
        __builtin_amdgcn_sched_barrier(0);
        if (GENERAL && t0 + TREE_KT > past)
        {
#pragma unroll
            for (int qt = 0; qt < QT; ++qt)
            {
                const int s0 = t0 - past; // > -64
                uint64_t seen;
                if (long_tree) // uniform
                {
                    const int node = min(q0 + 16 * qt + lr, n * G - 1) / G;
                    seen = tree_mask64(p.tree_mask + (size_t) (off + node) * p.mask_words, p.mask_words, n, s0);
                }
                else // the history's keys are seen
                    seen = s0 < 0 ? mask_row[qt] << -s0 | ((1ull << -s0) - 1) : (s0 < 64 ? mask_row[qt] >> s0 : 0);
                seen >>= kb0 + kb + 4 * lq;
#pragma unroll
                for (int x = 0; x < X2; ++x)
#pragma unroll
                    for (int rr = 0; rr < 4; ++rr)
                        s[x][qt][rr] = (seen >> (16 * x + rr)) & 1 ? s[x][qt][rr] : -__builtin_inff();
            }
        }
        uint32_t pk[QT][X2][2];
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
        {
            int mx = 0; // the largest positive s - m, as raw bits
#pragma unroll
            for (int x = 0; x < X2; ++x)
#pragma unroll
                for (int rr = 0; rr < 4; ++rr)
                    mx = max(mx, __builtin_bit_cast(int, (float) s[x][qt][rr]));
            const bool first = GENERAL && fresh[qt];
            if (__any(first || mx > GROWTH)) // wave-uniform
            {
                // the column's maximum of these keys, over its 4 lanes (a NaN stays out of the comparison and in the scores)
                float top = -__builtin_inff();
#pragma unroll
                for (int x = 0; x < X2; ++x)
#pragma unroll
                    for (int rr = 0; rr < 4; ++rr)
                        top = fmaxf(top, s[x][qt][rr]);
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                if (top != -__builtin_inff())
                {
                    // where fp32 counts in steps of 2 and more the maximum gets no lead, or P would leave fp16 by its rounding; below
                    // that the sums move by what the maximum moved by, rounding included
                    const bool coarse = fabsf(minus_m[qt][0] - top) >= 0x1p24f;
                    const float lead = coarse ? 0.f : LEAD;
                    float up = first ? top - lead : fmaxf(top - lead, 0.f);
                    const float mm = minus_m[qt][0] - up;
                    up = coarse ? up : minus_m[qt][0] - mm;
                    const float corr = first ? 0.f : __builtin_amdgcn_exp2f(-up); // (nothing was summed before the first maximum)
                    minus_m[qt] = cf32x4_t{mm, mm, mm, mm};
                    if constexpr (GENERAL)
                        fresh[qt] = false;
                    l_run[qt] *= corr;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                        for (int rr = 0; rr < 4; ++rr)
                            o[qt][dt][rr] *= corr;
#pragma unroll
                    for (int x = 0; x < X2; ++x)
#pragma unroll
                        for (int rr = 0; rr < 4; ++rr)
                            s[x][qt][rr] -= up;
                }
            }
#pragma unroll
            for (int x = 0; x < X2; ++x)
            {
                float e[4];
#pragma unroll
                for (int rr = 0; rr < 4; ++rr)
                {
                    e[rr] = __builtin_amdgcn_exp2f(s[x][qt][rr]);
                    l_run[qt] += e[rr];
                }
                // P in the compute type: its rounding (half a step, relative) averages out over the keys
                pk[qt][x][0] = pack2<C>(e[0], e[1]);
                pk[qt][x][1] = pack2<C>(e[2], e[3]);
            }
        }
        // ---- O^T += V^T . P^T  (A operand rows d = 16 dt + lr by the transposing LDS read)
#pragma unroll
        for (int d0 = 0; d0 < DT; d0 += VBATCH)
        {
            if (d0)
                read_v(d0);
#pragma unroll
            for (int dt = 0; dt < VBATCH; ++dt)
#pragma unroll
                for (int qt = 0; qt < QT; ++qt)
                {
                    if constexpr (X2 == 2)
                        o[qt][d0 + dt] = ctx_mfma<C>(make_uint4(vf[dt][0].x, vf[dt][0].y, vf[dt][X2 - 1].x, vf[dt][X2 - 1].y),
                            make_uint4(pk[qt][0][0], pk[qt][0][1], pk[qt][X2 - 1][0], pk[qt][X2 - 1][1]), o[qt][d0 + dt]);
                    else
                        o[qt][d0 + dt] = tree_mfma16<C>(vf[dt][0], make_uint2(pk[qt][0][0], pk[qt][0][1]), o[qt][d0 + dt]);
                }
        }
    };
    // V rows of a tile with nodes, in the LDS: rows past the sequence are zeroed (whatever lies there, 0 * NaN is NaN), and so
    // are nodes' elements that are not finite, which must not reach the columns that do not see them; the others get them
    // at the end.  History rows are seen by every column and stay as they are.
    auto clean_tail = [&](uint32_t stage, int t0)
    {
        for (int c = max(past - t0, 0) * CH + tid; c < TREE_KT * CH; c += TREE_THREADS)
        {
            const int row = c / CH, t = t0 + row;
            uint4* at = reinterpret_cast<uint4*>(lds + stage + TILE_BYTES + 16 * c);
            if (t >= total)
                *at = make_uint4(0, 0, 0, 0);
            else if (KVT == 0 && t >= past)
            {
                uint4 w = *at;
                uint32_t* x = reinterpret_cast<uint32_t*>(&w);
                if (tree_nonfinite2<T>(x[0]) || tree_nonfinite2<T>(x[1]) || tree_nonfinite2<T>(x[2]) || tree_nonfinite2<T>(x[3]))
                {
                    constexpr uint32_t EXP = T16<T>::is_bf16 ? 0x7f80u : 0x7c00u;
                    for (int e = 0; e < 4; ++e)
                    {
                        if ((x[e] & EXP) == EXP)
                            x[e] &= 0xffff0000u;
                        if (((x[e] >> 16) & EXP) == EXP)
                            x[e] &= 0xffffu;
                    }
                    *at = w;
                    atomicOr(&nonfinite[(t - past) >> 5], 1u << ((t - past) & 31));
                }
            }
        }
        __syncthreads();
    };

    uint32_t stage = 0; // of the tile that is computed
    int i = tile_lo;
    auto enter_tile = [&]()
    {
        if constexpr (KVT == 0)
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // my share of tile i has landed
        __syncthreads();                                     // everyone's has, and everyone is done with tile i - 1
        if (i + 1 < tile_hi)
        {
            load_tile(STAGE_BYTES - stage);
            find_tile(min(i + 2, tile_hi - 1));
        }
    };
    auto leave_tile = [&]()
    {
        stage = STAGE_BYTES - stage;
        ++i;
        if constexpr (KVT != 0)
        {
            if (i < tile_hi)
                store_tile(stage);
        }
    };
    // The first tile and the tiles with nodes go through the general step, the history's others through the short one: 328 us for 352
    // with the general step alone over 120001 tokens (60 nodes, 64 / 8 heads), 176 for 193 over 16 x 4096 in fp8.  Where the waves
    // share the keys one copy of the step is enough (16 nodes, 64 x 2048 tokens: 431 us either way).
    const bool has_rows = q0 < n * G; // a wave without rows (a smaller tree than the largest) only loads
    const int plain_end = KW == 1 ? min(tile_hi, past / TREE_KT) : 0;
    for (;; careful = true)
    {
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
        {
            fresh[qt] = true;
            l_run[qt] = 0.f;
            minus_m[qt] = cf32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
                o[qt][dt] = cf32x4_t{0.f, 0.f, 0.f, 0.f};
        }
        if constexpr (KVT != 0)
            store_tile(0);
        while (i < tile_hi)
        {
            enter_tile();
            const int t0 = i * TREE_KT;
            if (t0 + TREE_KT > past)
                clean_tail(stage, t0);
#pragma unroll 1
            for (int kb = has_rows ? 0 : 16 * XW; kb < 16 * XW; kb += 16 * X2)
                step(std::true_type{}, stage, kb, t0);
            leave_tile();
            if constexpr (KW == 1)
            {
                // (scores of -inf only, of an overflow in fp32: the column has no maximum yet, the general step goes on)
                bool open = careful;
#pragma unroll
                for (int qt = 0; qt < QT; ++qt)
                    open |= fresh[qt];
                const bool settled = !__any(open);
                while (settled && i < plain_end)
                {
                    enter_tile();
#pragma unroll 1
                    for (int kb = 0; kb < 16 * XW; kb += 16 * X2)
                        step(std::false_type{}, stage, kb, 0);
                    leave_tile();
                }
            }
        }
        bool bad = false;
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
            bad |= l_run[qt] != l_run[qt] || q_shift[qt] != 0;
        if (__any(bad))
            redo = 1;
        __syncthreads(); // (everyone is done with the tiles, too)
        if (careful || !__builtin_amdgcn_readfirstlane(redo))
            break;
        stage = 0;
        i = tile_lo;
        find_tile(tile_lo);
        load_tile(0);
        find_tile(min(tile_lo + 1, tile_hi - 1));
    }

    // ---- the end of the item: the sum over the 4 lanes of a column; the states of the KW key groups meet in the LDS, and
    // each of their waves joins and stores its share of the output columns
    constexpr int DTW = DT / KW;
    const int dt0 = kw * DTW;
    bool any_nonfinite = false;
    if constexpr (KVT == 0)
        for (int w = 0; w < (n + 31) >> 5; ++w)
            any_nonfinite |= nonfinite[w] != 0;
    const float v_deq = KVT ? p.kv_scale_quant_orig[0] : 1.f;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
    {
        float m = fresh[qt] ? TREE_NO_MAX : -minus_m[qt][0], l = l_run[qt];
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        cf32x4_t acc[DTW];
        if constexpr (KW == 1)
        {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
                acc[dt] = o[qt][dt];
        }
        else
        {
            constexpr int STATE = (DT + 1) * 64 * 16; // bytes of one wave's state: float4 per register group and lane
            static_assert(4 * STATE <= 2 * STAGE_BYTES, "states do not fit the tile buffers");
            if (qt > 0)
                __syncthreads(); // everyone is done with the states before
            cf32x4_t* st = reinterpret_cast<cf32x4_t*>(lds + wave * STATE) + lane;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
                st[dt * 64] = o[qt][dt];
            st[DT * 64] = cf32x4_t{m, l, 0.f, 0.f};
            __syncthreads();
            float c[KW], mk[KW], lk[KW];
#pragma unroll
            for (int k = 0; k < KW; ++k)
            {
                const cf32x4_t ml = reinterpret_cast<const cf32x4_t*>(lds + (k * RW + rw) * STATE)[DT * 64 + lane];
                mk[k] = ml[0];
                lk[k] = ml[1];
            }
            m = mk[0];
#pragma unroll
            for (int k = 1; k < KW; ++k)
                m = fmaxf(m, mk[k]);
            l = 0.f;
#pragma unroll
            for (int k = 0; k < KW; ++k)
            {
                c[k] = __builtin_amdgcn_exp2f(mk[k] - m);
                l += lk[k] * c[k];
            }
#pragma unroll
            for (int dt = 0; dt < DTW; ++dt)
            {
                acc[dt] = cf32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KW; ++k)
                {
                    const cf32x4_t x = reinterpret_cast<const cf32x4_t*>(lds + (k * RW + rw) * STATE)[(dt0 + dt) * 64 + lane];
#pragma unroll
                    for (int rr = 0; rr < 4; ++rr)
                        acc[dt][rr] += x[rr] * c[k];
                }
            }
        }
        const int in_tile = rw * QT * 16 + 16 * qt + lr, r = min(mt * M + in_tile, n * G - 1), node = r / G;
        if (any_nonfinite) // uniform, and rare
        {
            for (int j = 0; j < n; ++j)
            {
                if (!((nonfinite[j >> 5] >> (j & 31)) & 1))
                    continue;
                const int t = past + j;
                const size_t at = ((size_t) head_kv << p.tpb_log2) + (t & tpb_mask);
                const uint16_t* v = reinterpret_cast<const uint16_t*>(vp[t >> p.tpb_log2]) + at * hs;
                const bool sees = (p.tree_mask[(size_t) (off + node) * p.mask_words + (j >> 5)] >> (j & 31)) & 1;
#pragma unroll
                for (int dt = 0; dt < DTW; ++dt)
#pragma unroll
                    for (int rr = 0; rr < 4; ++rr)
                    {
                        const int d = 16 * (dt0 + dt) + 4 * lq + rr;
                        const uint32_t w = v[min(d, hs - 1)];
                        acc[dt][rr] += sees && d < hs && tree_nonfinite2<T>(w) ? T16<T>::to_float(w) : 0.f;
                    }
            }
        }
        if (mt * M + in_tile >= n * G)
            continue;
        if (parts == 1)
        {
            // no visible key: the sum is exactly 0, and so is the row (a NaN sum stays a NaN)
            const float inv = l == 0.f ? 0.f : v_deq / l;
            uint16_t* out = p.out + ((size_t) (off + node) * p.num_heads + head_kv * G + (r - node * G)) * hs;
#pragma unroll
            for (int dt = 0; dt < DTW; ++dt)
            {
                const int d = 16 * (dt0 + dt) + 4 * lq;
                if (d < hs)
                    *reinterpret_cast<uint2*>(out + d)
                        = make_uint2(pack2<T>(acc[dt][0] * inv, acc[dt][1] * inv), pack2<T>(acc[dt][2] * inv, acc[dt][3] * inv));
            }
        }
        else
        {
            const size_t rec = ((size_t) (__builtin_amdgcn_readlane(info_split.y, at) + in_seq) * p.mtiles + mt) * M + in_tile;
            float* part = p.part_acc + rec * DP;
#pragma unroll
            for (int dt = 0; dt < DTW; ++dt)
                *reinterpret_cast<cf32x4_t*>(part + 16 * (dt0 + dt) + 4 * lq) = acc[dt];
            if (lq == 0 && kw == 0)
                p.part_ml[rec] = make_float2(m, l);
        }
    }
}

// ---------------------------------------------------------------------------------------------- 3. combine
// grid (ceil(rows of a (sequence, kv head) / 8), pairs of several parts at most).  Half a wave joins one row; the parts are summed in
// the keys' order, 4 in flight.  Bound by the reads of the states: 8.5 us for 18 MB (256 pairs of 20 .. 108 rows), 4.2 us at least.
template <typename T, int DP>
__global__ __launch_bounds__(TREE_THREADS) void tree_combine_kernel(TreeArgs p, bool quantised)
{
    const int lane = threadIdx.x & 31;
    const int4 join = p.join[2 * blockIdx.y], where = p.join[2 * blockIdx.y + 1];
    const int S = join.w, G = p.group, r = blockIdx.x * (TREE_THREADS / 32) + (threadIdx.x >> 5);
    if (S <= 1 || r >= join.y * G || !p.seq_ok[where.y])
        return;
    const int M = p.rows_per_wg;
    auto record = [&](int s) { return ((size_t) (where.x + s) * p.mtiles + r / M) * M + r % M; };
    constexpr int E = DP / 32, U = 4;
    float mm = TREE_NO_MAX, l = 0.f;
    for (int s = lane; s < S; s += 32)
        mm = fmaxf(mm, p.part_ml[record(s)].x);
#pragma unroll
    for (int x = 16; x >= 1; x >>= 1)
        mm = fmaxf(mm, __shfl_xor(mm, x));
    float acc[E] = {};
    for (int s0 = 0; s0 < S; s0 += U)
    {
        float v[U][E];
        float2 ml[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
        {
            const size_t rec = record(min(s0 + u, S - 1));
            ml[u] = p.part_ml[rec];
#pragma unroll
            for (int e = 0; e < E; ++e)
                v[u][e] = p.part_acc[rec * DP + E * lane + e];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s0 + u < S)
            {
                const float c = __builtin_amdgcn_exp2f(ml[u].x - mm);
                l += ml[u].y * c;
#pragma unroll
                for (int e = 0; e < E; ++e)
                    acc[e] += v[u][e] * c;
            }
    }
    const float inv = l == 0.f ? 0.f : (quantised ? p.kv_scale_quant_orig[0] : 1.f) / l;
    uint16_t* out = p.out + ((size_t) (join.x + r / G) * p.num_heads + join.z * G + r % G) * p.hs + E * lane;
#pragma unroll
    for (int e = 0; e < E; e += 2)
        if (E * lane + e < p.hs)
            *reinterpret_cast<uint32_t*>(out + e) = pack2<T>(acc[e] * inv, acc[e + 1] * inv);
}

// ---------------------------------------------------------------------------------------------- host
struct TreePlan
{
    int dp, rows_per_wg, mtiles; // padded head size; query rows per workgroup; m-tiles of a (sequence, kv head)
    int target_items, part_tiles, items_bound, pairs_bound, records, whole;
    size_t q_bytes, shift_bytes, order_bytes, split_bytes, ok_bytes, join_bytes, acc_bytes, ml_bytes;
    size_t total() const
    {
        return q_bytes + shift_bytes + order_bytes + split_bytes + ok_bytes + join_bytes + acc_bytes + ml_bytes;
    }
};
size_t round256(size_t x)
{
    return (x + 255) / 256 * 256;
}

void tree_check(const mi355q_tree_attention_params& q)
{
    MQ_CHECK(q.act_type == MI355Q_HALF || q.act_type == MI355Q_BF16, "act_type %d", q.act_type);
    MQ_CHECK(q.kv_type == q.act_type || q.kv_type == MI355Q_INT8 || q.kv_type == MI355Q_FP8, "kv cache type %d", q.kv_type);
    MQ_CHECK(q.batch >= 0 && q.batch <= 65535 && q.num_heads > 0 && q.num_kv_heads > 0 && q.num_heads % q.num_kv_heads == 0,
        "batch %d, heads %d / %d", q.batch, q.num_heads, q.num_kv_heads);
    MQ_CHECK(q.head_size >= 8 && q.head_size <= 256 && q.head_size % (q.kv_type == q.act_type ? 8 : 16) == 0,
        "tree attention: head_size %d (multiples of 8, with an 8-bit cache of 16, up to 256)", q.head_size);
    MQ_CHECK(q.num_tokens >= 0 && q.max_draft_length >= 0 && q.max_draft_length <= TREE_MAX_DRAFT,
        "num_tokens %d, max_draft_length %d (at most %d)", q.num_tokens, q.max_draft_length, TREE_MAX_DRAFT);
    MQ_CHECK((int64_t) q.num_heads * q.max_draft_length <= (1 << 24), "num_heads %d x max_draft_length %d", q.num_heads, q.max_draft_length);
    MQ_CHECK(q.tokens_per_block > 0 && (q.tokens_per_block & (q.tokens_per_block - 1)) == 0 && q.tokens_per_block <= (1 << 20),
        "tokens_per_block must be a power of 2, got %d", q.tokens_per_block);
    if (q.tokens_per_block < 16) // a wave's 16 keys of a tile come from one block
        MQ_UNSUPPORTED("tree attention: tokens_per_block %d is not built (16 or more)", q.tokens_per_block);
    MQ_CHECK(q.max_blocks_per_seq > 0, "max_blocks_per_seq %d", q.max_blocks_per_seq);
    MQ_CHECK(q.max_past_length >= 0 && q.max_past_length <= (1 << 30), "max_past_length %d", q.max_past_length);
    MQ_CHECK(q.multi_block_mode >= 0, "multi_block_mode %d", q.multi_block_mode);
}

TreePlan tree_plan(const mi355q_tree_attention_params& q)
{
    TreePlan t{};
    t.dp = q.head_size <= 64 ? 64 : (q.head_size <= 128 ? 128 : 256);
    const int rows = std::max(q.max_draft_length, 1) * (q.num_heads / q.num_kv_heads);
    const int max_tiles = std::max((q.max_past_length + q.max_draft_length + TREE_KT - 1) / TREE_KT, 1);
    const int64_t groups = (int64_t) q.batch * q.num_kv_heads;
    // Few rows: the 4 waves of a workgroup share the keys of a tile instead of the rows.  Whole calls, us, with 16 / 32 / 64 / 128 rows
    // a workgroup (bf16, Dh 128, 32 sequences of 2048 tokens, 32 heads): 16 nodes 230 / 230 / 232 / 233, 32 nodes 262 / 238 / 242 /
    // 243, 64 nodes 403 / 291 / 270 / 275, 128 nodes 718 / 453 / 356 / 334.
    // 33 to 64 rows of fewer than 256 (sequence, kv head) pairs go as two tiles of 32: half as many parts, so fewer states to
    // join (8 nodes x 8 heads over 4096 tokens, 4 / 8 / 16 / 32 sequences: 29.2 / 37.3 / 61.0 / 128 us, as one tile of 64 33.8 / 41.8 /
    // 64.3 / 127)
    t.rows_per_wg = rows <= 16 ? 16 : (rows <= 32 || (rows <= 64 && t.dp <= 128 && groups < 256) ? 32 : (rows <= 64 || t.dp > 128 ? 64 : 128));
    t.mtiles = (rows + t.rows_per_wg - 1) / t.rows_per_wg;
    // One item per (sequence, kv head), nothing to join, for short histories: up to 512 keys, and up to 4096 tokens of history the
    // longer the more workgroups there are to even the lengths out (64 tiles with the chip's 512; the nodes on top of a history do
    // not count, or 4096 tokens would be cut).  us whole / in parts, equal histories of t tokens: 8 workgroups (one sequence, 8 kv heads, 8
    // nodes) t = 512 16.8 / 15.9; 32 (32 kv heads) 440 13.2 / 15.0, 512 15.5 / 15.9, 1000 18.4 / 16.1; 128 (4 sequences, 16 nodes) 600 19.0 /
    // 22.9, 1024 24.4 / 27.5 (ragged 23.2 / 24.3); 256 (8) 2048 51.4 / 58.0 (ragged 40.9 / 44.5), 3400 101.2 / 100.6 (ragged 66.0 /
    // 60.3); 512 (16, 64 nodes, 64 / 8 heads) 4096 190.1 / 192.1 (ragged 126.9 / 130.0), fp8 155.5 / 156.8 (ragged 116.8 / 119.4); 1024 (32)
    // 4100 417 / 430
    const int history_tiles = (q.max_past_length + TREE_KT - 1) / TREE_KT;
    const int64_t whole_tiles = std::min<int64_t>(groups * t.mtiles / 8, 64);
    t.whole = q.multi_block_mode == 1 || (q.multi_block_mode == 0 && (max_tiles <= 8 || history_tiles <= whole_tiles));
    if (t.whole)
        t.items_bound = (int) std::min<int64_t>(groups, INT32_MAX / 16);
    else if (q.multi_block_mode > 0)
    {
        // that many parts of the longest history
        const int splits = std::min({q.multi_block_mode, max_tiles, TREE_MAX_SPLITS});
        t.part_tiles = -((max_tiles + splits - 1) / splits);
        t.items_bound = (int) std::min<int64_t>(groups * splits, INT32_MAX / 16);
        t.pairs_bound = (int) std::min<int64_t>(groups, t.items_bound / 2);
        t.records = t.items_bound;
    }
    else
    {
        // two workgroups live on a CU (one with heads beyond 128): about as many items as fill 256 CUs, of at least 2 tiles each (an
        // item costs its prologue and a partial state; 512 / 1024 items, us: 4 sequences of 4000 tokens, 8 nodes, 32 / 8 heads 28 / 35,
        // 16 of 4100, 64 nodes, 64 / 8 heads 212 / 230, ragged 132 / 139), and no pair in more parts than the combine kernel reads.  A pair of nt
        // tiles has round(nt / part) parts where that is 2 or more: at most 4 / 3 nt / part
        t.target_items = std::max((t.dp > 128 ? 256 : 512) / t.mtiles, 1);
        t.part_tiles = std::max(2, (max_tiles + TREE_MAX_SPLITS - 1) / TREE_MAX_SPLITS);
        t.records = t.target_items + t.target_items / 3 + 1;
        t.pairs_bound = (int) std::min<int64_t>(groups, t.records / 2);
        t.items_bound = (int) std::min<int64_t>(groups + t.records, INT32_MAX / 16);
    }
    const bool two_parts = q.kv_type == q.act_type || q.act_type == MI355Q_HALF; // TREE_Q2
    t.q_bytes = round256((size_t) q.num_tokens * q.num_heads * t.dp * 2 * (two_parts ? 2 : 1));
    if (q.act_type == MI355Q_HALF || q.kv_type != q.act_type) // products in fp16
        t.shift_bytes = round256((size_t) q.num_tokens * q.num_heads);
    t.order_bytes = round256((size_t) (q.batch + 1) * sizeof(int4));
    t.split_bytes = round256((size_t) q.batch * sizeof(int4));
    t.ok_bytes = round256((size_t) q.batch * sizeof(int32_t));
    if (!t.whole)
    {
        t.join_bytes = round256((size_t) t.pairs_bound * 2 * sizeof(int4));
        const size_t records = (size_t) t.records * t.mtiles * t.rows_per_wg;
        t.acc_bytes = round256(records * t.dp * sizeof(float));
        t.ml_bytes = round256(records * sizeof(float2));
    }
    return t;
}

template <typename T, int KVT, int DP>
void tree_launch_attn(const TreeArgs& a, const TreePlan& t, hipStream_t stream)
{
    const int64_t grid = ((int64_t) t.items_bound + 7) / 8 * 8 * t.mtiles;
    const dim3 g((unsigned) grid), b(TREE_THREADS);
    // 32 rows a wave; 16 with heads beyond 128, whose accumulators take twice the registers
    constexpr int QT = DP > 128 ? 1 : 2;
    if (t.rows_per_wg == 16)
        hipLaunchKernelGGL((tree_attn_kernel<T, KVT, DP, 1, 4, 1>), g, b, 0, stream, a);
    else if (t.rows_per_wg == 32)
        hipLaunchKernelGGL((tree_attn_kernel<T, KVT, DP, 2, 2, 1>), g, b, 0, stream, a);
    else if (t.rows_per_wg == 32 * QT)
        hipLaunchKernelGGL((tree_attn_kernel<T, KVT, DP, 2, 2, QT>), g, b, 0, stream, a);
    else
        hipLaunchKernelGGL((tree_attn_kernel<T, KVT, DP, 4, 1, QT>), g, b, 0, stream, a);
    MQ_HIP(hipGetLastError());
}

template <typename T, int KVT>
void tree_launch(const mi355q_tree_attention_params& q, const TreeArgs& a, const TreePlan& t, hipStream_t stream)
{
    // a token's heads over several workgroups, one 8-element chunk a thread, while the tokens alone do not fill the chip
    const int passes = ((q.num_heads + 2 * q.num_kv_heads) * t.dp / 8 + TREE_THREADS - 1) / TREE_THREADS;
    const int parts = std::max(1, (int) std::min<int64_t>(passes, 2048 / ((int64_t) q.batch * q.max_draft_length)));
    hipLaunchKernelGGL((tree_prepare_kernel<T, KVT>), dim3(q.max_draft_length + 2, q.batch, parts), dim3(TREE_THREADS), 0, stream, a, t.dp);
    MQ_HIP(hipGetLastError());
    if (t.dp == 64)
        tree_launch_attn<T, KVT, 64>(a, t, stream);
    else if (t.dp == 128)
        tree_launch_attn<T, KVT, 128>(a, t, stream);
    else
        tree_launch_attn<T, KVT, 256>(a, t, stream);
    if (!t.whole && t.pairs_bound)
    {
        const dim3 g((t.mtiles * t.rows_per_wg + 7) / 8, t.pairs_bound), b(TREE_THREADS);
        if (t.dp == 64)
            hipLaunchKernelGGL((tree_combine_kernel<T, 64>), g, b, 0, stream, a, KVT != 0);
        else if (t.dp == 128)
            hipLaunchKernelGGL((tree_combine_kernel<T, 128>), g, b, 0, stream, a, KVT != 0);
        else
            hipLaunchKernelGGL((tree_combine_kernel<T, 256>), g, b, 0, stream, a, KVT != 0);
        MQ_HIP(hipGetLastError());
    }
}

template <typename T>
void tree_launch_kv(const mi355q_tree_attention_params& q, const TreeArgs& a, const TreePlan& t, hipStream_t stream)
{
    if (q.kv_type == q.act_type)
        tree_launch<T, 0>(q, a, t, stream);
    else if (q.kv_type == MI355Q_INT8)
        tree_launch<T, 1>(q, a, t, stream);
    else
        tree_launch<T, 2>(q, a, t, stream);
}

bool aligned16(const void* p)
{
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}
} // namespace

size_t tree_attention_workspace_size(const mi355q_tree_attention_params& q)
{
    tree_check(q);
    return tree_plan(q).total();
}

void tree_attention(const mi355q_tree_attention_params& q, hipStream_t stream)
{
    tree_check(q);
    if (q.batch == 0 || q.num_tokens == 0 || q.max_draft_length == 0)
        return;
    const size_t hidden = (size_t) (q.num_heads + 2 * q.num_kv_heads) * q.head_size;
    MQ_CHECK(q.qkv && q.out && q.past_lengths && q.draft_offsets && q.tree_mask && q.block_pointers, "null tensor");
    MQ_CHECK(q.qkv_stride == 0 || ((size_t) q.qkv_stride >= hidden && q.qkv_stride % 8 == 0), "qkv_stride %lld (rows of %zu)",
        (long long) q.qkv_stride, hidden);
    MQ_CHECK(aligned16(q.qkv) && aligned16(q.qkv_bias) && aligned16(q.out) && aligned16(q.workspace), "tensors must be 16-byte aligned");
    MQ_CHECK(q.mask_words >= (q.max_draft_length + 31) / 32, "tree_mask rows of %d words do not hold %d nodes", q.mask_words,
        q.max_draft_length);
    MQ_CHECK((int64_t) q.max_past_length <= (int64_t) q.max_blocks_per_seq * q.tokens_per_block,
        "past length %d exceeds the block table (%d x %d)", q.max_past_length, q.max_blocks_per_seq, q.tokens_per_block);
    if (q.kv_type != q.act_type)
        MQ_CHECK(q.kv_scale_orig_quant && q.kv_scale_quant_orig, "8-bit kv cache needs kv_scale_orig_quant and kv_scale_quant_orig");
    if (q.position_embedding_type == 1 || q.position_embedding_type == 2)
    {
        MQ_CHECK(q.rotary_embedding_dim > 0 && q.rotary_embedding_dim <= q.head_size && q.rotary_embedding_dim % 2 == 0,
            "rotary_embedding_dim %d", q.rotary_embedding_dim);
        MQ_CHECK(q.rotary_embedding_base > 0.f, "rotary_embedding_base %g", q.rotary_embedding_base);
        MQ_CHECK(q.rotary_embedding_scale_type >= 0 && q.rotary_embedding_scale_type <= 2, "rotary_embedding_scale_type %d",
            q.rotary_embedding_scale_type);
        if (q.rotary_embedding_scale_type != 0)
            MQ_CHECK(q.rotary_embedding_scale > 0.f, "rotary_embedding_scale %g", q.rotary_embedding_scale);
        if (q.rotary_embedding_scale_type == 2)
            MQ_CHECK(q.rotary_embedding_max_positions > 0 && q.rotary_embedding_dim > 2 && q.rotary_embedding_scale >= 1.f,
                "dynamic rotary scaling: max_positions %d, dim %d, scale %g", q.rotary_embedding_max_positions, q.rotary_embedding_dim,
                q.rotary_embedding_scale);
    }
    else if (q.position_embedding_type != 0)
        MQ_UNSUPPORTED("tree attention: position_embedding_type %d is not built (0 - 2)", q.position_embedding_type);
    const TreePlan t = tree_plan(q);
    MQ_CHECK((int64_t) q.batch * q.num_kv_heads * ((q.max_past_length + q.max_draft_length + TREE_KT - 1) / TREE_KT) < (1 << 30),
        "tree attention: %d sequences x %d kv heads x %d keys", q.batch, q.num_kv_heads, q.max_past_length);
    // what the grids hold (2^32 threads, 65535 rows)
    MQ_CHECK(((int64_t) t.items_bound + 8) * t.mtiles < (1ll << 24) && t.pairs_bound <= 65535,
        "tree attention: %d sequences x %d kv heads x %d row tiles, up to %d pairs in parts", q.batch, q.num_kv_heads, t.mtiles, t.pairs_bound);
    MQ_CHECK(q.workspace && q.workspace_bytes >= t.total(), "workspace too small: %zu < %zu", q.workspace_bytes, t.total());
    TreeArgs a{};
    a.qkv = static_cast<const uint16_t*>(q.qkv);
    a.qkv_bias = static_cast<const uint16_t*>(q.qkv_bias);
    a.out = static_cast<uint16_t*>(q.out);
    a.past_lengths = q.past_lengths;
    a.draft_offsets = q.draft_offsets;
    a.position_offsets = q.position_offsets;
    a.tree_mask = q.tree_mask;
    a.block_ptrs = q.block_pointers;
    a.kv_scale_orig_quant = q.kv_scale_orig_quant;
    a.kv_scale_quant_orig = q.kv_scale_quant_orig;
    char* ws = static_cast<char*>(q.workspace);
    auto carve = [&](size_t bytes)
    {
        char* at = ws;
        ws += bytes;
        return at;
    };
    a.q_ws = reinterpret_cast<uint16_t*>(carve(t.q_bytes));
    a.q_shift = reinterpret_cast<uint8_t*>(carve(t.shift_bytes));
    a.order = reinterpret_cast<int4*>(carve(t.order_bytes));
    a.split = reinterpret_cast<int4*>(carve(t.split_bytes));
    a.seq_ok = reinterpret_cast<int32_t*>(carve(t.ok_bytes));
    a.join = reinterpret_cast<int4*>(carve(t.join_bytes));
    a.part_acc = reinterpret_cast<float*>(carve(t.acc_bytes));
    a.part_ml = reinterpret_cast<float2*>(carve(t.ml_bytes));
    a.qkv_stride = q.qkv_stride ? q.qkv_stride : (int64_t) hidden;
    a.batch = q.batch;
    a.num_heads = q.num_heads;
    a.num_kv_heads = q.num_kv_heads;
    a.group = q.num_heads / q.num_kv_heads;
    a.hs = q.head_size;
    a.num_tokens = q.num_tokens;
    a.max_draft = q.max_draft_length;
    a.max_past = q.max_past_length;
    a.mask_words = q.mask_words;
    a.max_blocks = q.max_blocks_per_seq;
    while ((1 << a.tpb_log2) < q.tokens_per_block)
        ++a.tpb_log2;
    a.mtiles = t.mtiles;
    a.rows_per_wg = t.rows_per_wg;
    a.target_items = t.target_items;
    a.part_tiles = t.part_tiles;
    a.items_bound = t.items_bound;
    a.pairs_bound = t.pairs_bound;
    a.whole = t.whole;
    a.pos_type = q.position_embedding_type;
    a.rot_dim = q.rotary_embedding_dim;
    a.rot_scale_type = q.rotary_embedding_scale_type;
    a.rot_max_pos = q.rotary_embedding_max_positions;
    a.rot_log2_base = q.rotary_embedding_base > 0.f ? log2((double) q.rotary_embedding_base) : 0.0;
    a.rot_scale = q.rotary_embedding_scale;
    a.score_scale = 1.f / (sqrtf((float) q.head_size) * (q.q_scaling == 0.f ? 1.f : q.q_scaling));
    if (q.act_type == MI355Q_BF16)
        tree_launch_kv<bf16_t>(q, a, t, stream);
    else
        tree_launch_kv<f16_t>(q, a, t, stream);
}

} // namespace mi355q
