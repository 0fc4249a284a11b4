// extern "C" entries of attention (declared in include/dlf_b200.h): argument checks, the choice of the kernel, tensor maps
// and launches.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <mutex>

#include "../../include/dlf_b200.h"
#include "attention_decode.cuh"
#include "attention_plan.h"
#include "attention_short.cuh"
#include "attention_tiles.cuh"
#include "host.cuh"

using namespace dlfb200;

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kDecodeLeast = 2;    // units a CTA takes at least
constexpr int kB200Sms = 148;  // for sizes that are asked for without a device at hand

struct AttentionDevice {
    bool ready = false;
};
AttentionDevice g_attention[kMaxDevices];
std::mutex g_attention_mu;

template <bool BF16, int DP>
int attention_limits() {
    for (auto k : {attention_decode_kernel<BF16, DP, KEYS_PLAIN, 1, true>, attention_decode_kernel<BF16, DP, KEYS_PLAIN, 1, false>,
                   attention_decode_kernel<BF16, DP, KEYS_PAGES_16, 1, true>, attention_decode_kernel<BF16, DP, KEYS_ANY, 1, true>,
                   attention_decode_kernel<BF16, DP, KEYS_ANY, 1, false>})
        CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, decode_smem(DP, 1)));
    for (auto k : {attention_decode_kernel<BF16, DP, KEYS_PLAIN, 2, true>, attention_decode_kernel<BF16, DP, KEYS_PLAIN, 2, false>,
                   attention_decode_kernel<BF16, DP, KEYS_PAGES_16, 2, true>, attention_decode_kernel<BF16, DP, KEYS_ANY, 2, true>,
                   attention_decode_kernel<BF16, DP, KEYS_ANY, 2, false>})
        CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, decode_smem(DP, 2)));
    CUDA_TRY(cudaFuncSetAttribute(attention_short_kernel<BF16, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, short_smem(DP, kTileKeys, 2)));
    CUDA_TRY(cudaFuncSetAttribute(attention_tiles_kernel<BF16, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, tiles_smem(DP)));
    return kSuccess;
}

int attention_device(const OperatorDevice& dev) {
    std::lock_guard<std::mutex> lock(g_attention_mu);
    AttentionDevice& st = g_attention[dev.device];
    if (st.ready) return kSuccess;
    for (int rc : {attention_limits<false, 64>(), attention_limits<false, 128>(), attention_limits<true, 64>(), attention_limits<true, 128>()})
        if (rc != kSuccess) return rc;
    st.ready = true;
    return kSuccess;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool scale_ok(float scale) { return scale > 0.0f && !std::isinf(scale * kLog2e); }
// strides that 16-byte pieces and tensor maps take
bool strides_ok(std::initializer_list<size_t> s) {
    for (size_t x : s)
        if (x % 8 != 0 || x >= (1ull << 38)) return false;
    return true;
}

// A workspace may start anywhere; the parts in it, read and written in pieces of 16 bytes, start at the next multiple of 256.
constexpr size_t kWorkspaceRoom = 256;
float* workspace_parts(void* workspace) {
    return reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(workspace) + kWorkspaceRoom - 1) / kWorkspaceRoom * kWorkspaceRoom);
}
// (sequences of one tile of keys are never cut)
size_t tiles_workspace(size_t keys, size_t size) {
    return keys > kTileKeys ? static_cast<size_t>(2 * kB200Sms) * tiles_slot(static_cast<int>(size)) * 4 + kWorkspaceRoom : 0;
}
size_t decode_workspace(size_t size) {
    const size_t ctas = static_cast<size_t>(kB200Sms * decode_ctas_per_sm(static_cast<int>(size), 1));
    return ctas * (2 * decode_slot(static_cast<int>(size)) * sizeof(float) + sizeof(int4)) + kWorkspaceRoom;
}

template <bool BF16, int DP, int KEYS, int NB, bool FULL>
int decode_launch(const DecodeParams& p, cudaStream_t stream) {
    CUDA_TRY(launch_dependent(attention_decode_kernel<BF16, DP, KEYS, NB, FULL>, static_cast<unsigned>(p.ctas), kDecodeThreads, decode_smem(DP, NB), stream, p));
    count_launch();
    // CTAs that may have work, of which the last cuts nothing; a sequence of one unit is never cut
    const long long units = plan_units(p.keys, kDecodeUnit), all = units * p.batch * p.kv_heads * p.row_blocks;
    const long long busy = std::min<long long>(p.ctas, (all + p.least - 1) / p.least);
    if (units > 1 && busy > 1) {
        CUDA_TRY(launch_dependent(attention_join_kernel<BF16>, static_cast<unsigned>(busy - 1), 128u, 0, stream, p));
        count_launch();
    }
    CUDA_TRY(cudaGetLastError());
    return kSuccess;
}
template <bool BF16, int DP, int NB>
int decode_keys(const DecodeParams& p, cudaStream_t stream) {
    const bool full = p.size == DP;
    if (p.table != nullptr && full && p.page_size % 16 == 0) return decode_launch<BF16, DP, KEYS_PAGES_16, NB, true>(p, stream);
    if (p.table != nullptr || p.mask != nullptr)
        return full ? decode_launch<BF16, DP, KEYS_ANY, NB, true>(p, stream) : decode_launch<BF16, DP, KEYS_ANY, NB, false>(p, stream);
    return full ? decode_launch<BF16, DP, KEYS_PLAIN, NB, true>(p, stream) : decode_launch<BF16, DP, KEYS_PLAIN, NB, false>(p, stream);
}
template <bool BF16, int DP>
int decode_rows(DecodeParams& p, cudaStream_t stream) {
    const int rows = p.tokens * p.group;
    p.block_rows = rows <= 8 ? 8 : 16;
    p.ctas *= decode_ctas_per_sm(DP, rows <= 8 ? 1 : 2);
    p.cuts = reinterpret_cast<int4*>(p.parts + 2ll * p.ctas * decode_slot(p.size));
    p.row_blocks = (rows + p.block_rows - 1) / p.block_rows;
    return rows <= 8 ? decode_keys<BF16, DP, 1>(p, stream) : decode_keys<BF16, DP, 2>(p, stream);
}
int decode_any(DecodeParams& p, bool bf16, cudaStream_t stream) {
    if (p.size <= 64) return bf16 ? decode_rows<true, 64>(p, stream) : decode_rows<false, 64>(p, stream);
    return bf16 ? decode_rows<true, 128>(p, stream) : decode_rows<false, 128>(p, stream);
}

// tensor map of a (batch, tokens, heads, size) tensor: boxes of `rows` tokens x 64 (or 32) values of one head, swizzled by 128 (64) bytes
int encode_heads(const OperatorDevice& dev, CUtensorMap* map, const void* base, size_t size, size_t tokens, size_t heads, size_t batch,
                 size_t st, size_t sh, size_t sb, unsigned rows, unsigned values = 64) {
    auto stride = [](size_t extent, size_t s) { return static_cast<cuuint64_t>(extent > 1 && s > 0 ? s * 2 : 16); };
    cuuint64_t dims[4] = {size, tokens, heads, sb == 0 ? 1 : batch};
    cuuint64_t strides[3] = {stride(tokens, st), stride(heads, sh), stride(dims[3], sb)};
    cuuint32_t box[4] = {values, rows, 1, 1}, estr[4] = {1, 1, 1, 1};
    const CUresult r = dev.encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, const_cast<void*>(base), dims, strides, box, estr,
                                  CU_TENSOR_MAP_INTERLEAVE_NONE, values == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? kSuccess : kUnexpectedError;
}

template <bool BF16, int DP>
int tiles_launch(const TilesParams& p, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& y, cudaStream_t stream) {
    CUDA_TRY(launch_dependent(attention_tiles_kernel<BF16, DP>, static_cast<unsigned>(p.ctas), kTilesThreads, tiles_smem(DP), stream, p, q, k, v, y));
    count_launch();
    if (p.ctas > 1) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<unsigned>(p.ctas - 1), 256 / kTilesJoinRows, 1);
        cfg.blockDim = dim3(128, 1, 1);
        cfg.stream = stream;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        CUDA_TRY(cudaLaunchKernelEx(&cfg, attention_tiles_join_kernel<BF16>, p));
        count_launch();
    }
    CUDA_TRY(cudaGetLastError());
    return kSuccess;
}

template <bool BF16, int DP>
int short_launch(ShortParams& p, int num_sms, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& y, cudaStream_t stream) {
    // The next tile's queries in a buffer of their own, unless that leaves one block to an SM (heads of 128 over more than 80 keys:
    // 16 x 4096 queries over 112, 8 heads, 84 us with one buffer and two blocks, 92 with two and one); not for a fourth block (heads
    // of 64 over more than 80: 35.6 us over 96 keys with three blocks of two buffers, 38.4 with four of one).
    auto per_sm_with = [&](int buffers) { return std::min(short_ctas_per_sm(DP), 228 * 1024 / (short_smem(DP, p.key_rows, buffers) + 1280)); };
    p.buffers = per_sm_with(2) < 2 ? 1 : 2;
    const int per_sm = per_sm_with(p.buffers), smem = short_smem(DP, p.key_rows, p.buffers);
    CUDA_TRY(launch_dependent(attention_short_kernel<BF16, DP>, static_cast<unsigned>(std::min(p.tiles, num_sms * per_sm)), kShortThreads, smem, stream, p, q, k, v, y));
    count_launch();
    CUDA_TRY(cudaGetLastError());
    return kSuccess;
}

// Few queries: the kernel that runs through the keys for 16 rows (a token's heads of a group are rows too). It does as much work as
// there are rows, the other one as if every head had 128 queries at least; with 32 entries of 1500 keys and 8 heads, one to a kv head (us, this
// kernel and the other): heads of 64 24 and 47 (16 queries), 33 and 47 (32), 53 and 48 (64); heads of 128 45 and 59 (16), 73 and
// 60 (32). 32 query heads on one kv head, 1 query: 13 and 128.
// Over up to 128 keys the other one is attention_short_kernel, and 8 queries are few: 256 entries of 77 keys, 8 heads (us), heads of
// 64 17 and 19 (8 queries), 23 and 19 (16), 44 and 19 (32); heads of 128 25 and 30 (8), 40 and 31 (16).
bool few_rows(size_t queries, size_t keys, size_t size) { return queries <= (keys <= kTileKeys ? 8 : size <= 64 ? 32 : 16); }

int head_args(int dtype, size_t heads, size_t kv_heads, size_t size) {
    if (dtype != DLF_B200_HALF && dtype != DLF_B200_BFLOAT16) return kNotImplemented;
    if (heads == 0 || kv_heads == 0 || size == 0 || heads % kv_heads != 0 || heads > 65535) return kInvalidDimension;
    if (size > 128 || size % 8 != 0) return kNotImplemented;
    return kSuccess;
}

}  // namespace

extern "C" {

size_t dlf_b200_attention_workspace_bytes(size_t batch, size_t queries, size_t keys, size_t heads, size_t kv_heads, size_t size) {
    (void)batch;
    if (kv_heads == 0 || heads % kv_heads != 0) return 0;
    return few_rows(queries, keys, size) ? decode_workspace(size) : tiles_workspace(keys, size);
}

int dlf_b200_attention(const dlf_b200_attention_args* args, void* workspace, size_t workspace_bytes, void* stream) {
    if (args == nullptr) return kInvalidValue;
    const auto& [dtype, scale, batch, queries, keys, heads, kv_heads, size, q_strides, k_strides, v_strides, y_strides, key_mask_ld, q, k, v, y,
                 key_lengths, key_mask] = *args;
    int rc = head_args(dtype, heads, kv_heads, size);
    if (rc != kSuccess) return rc;
    if (batch == 0 || queries == 0 || keys == 0 || batch > 65535 || queries > INT_MAX / 2 || keys > INT_MAX / 2) return kInvalidDimension;
    if (!scale_ok(scale)) return kInvalidValue;
    if (q == nullptr) return kInvalidMatrixA;
    if (k == nullptr || v == nullptr) return kInvalidMatrixB;
    if (y == nullptr) return kInvalidMatrixC;
    if (key_mask != nullptr && key_mask_ld < keys && key_mask_ld != 0 && batch > 1) return kInvalidLeadDimB;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(y) ||
        !strides_ok({q_strides[0], q_strides[1], q_strides[2], k_strides[0], k_strides[1], k_strides[2], v_strides[0], v_strides[1], v_strides[2],
                     y_strides[0], y_strides[1], y_strides[2]}))
        return kNotImplemented;
    if ((batch > 1 && y_strides[0] == 0) || (queries > 1 && y_strides[1] == 0) || (heads > 1 && y_strides[2] == 0)) return kInvalidLeadDimC;
    if ((queries > 1 && q_strides[1] == 0) || (heads > 1 && q_strides[2] == 0)) return kInvalidLeadDimA;
    if ((keys > 1 && (k_strides[1] == 0 || v_strides[1] == 0)) || (kv_heads > 1 && (k_strides[2] == 0 || v_strides[2] == 0))) return kInvalidLeadDimB;
    const bool bf16 = dtype == DLF_B200_BFLOAT16;
    const size_t group = heads / kv_heads;
    const bool few = few_rows(queries, keys, size);
    const size_t need = dlf_b200_attention_workspace_bytes(batch, queries, keys, heads, kv_heads, size);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return kInsufficientMemoryTemp;
    const long long items = static_cast<long long>((queries + 255) / 256) * static_cast<long long>(heads) * static_cast<long long>(batch);
    if (static_cast<double>(items) * (static_cast<double>(keys) / kTileKeys + 1.0) > 2147483647.0 || 2.0 * static_cast<double>(batch) * heads * (keys / kDecodeUnit + 1.0) > 2147483647.0) return kInvalidDimension;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    StreamDevice guard(s);
    if (guard.rc != kSuccess) return guard.rc;
    OperatorDevice dev;
    rc = operator_device(&dev);
    if (rc != kSuccess) return rc;
    rc = attention_device(dev);
    if (rc != kSuccess) return rc;
    clear_stale_error();
    const float c = scale * kLog2e;
    if (few) {
        DecodeParams p{};
        p.q = static_cast<const char*>(q);
        p.k = static_cast<const char*>(k);
        p.v = static_cast<const char*>(v);
        p.y = static_cast<char*>(y);
        p.q_sb = q_strides[0], p.q_st = q_strides[1], p.q_sh = q_strides[2];
        p.k_sb = k_strides[0], p.k_st = k_strides[1], p.k_sh = k_strides[2];
        p.v_sb = v_strides[0], p.v_st = v_strides[1], p.v_sh = v_strides[2];
        p.y_sb = y_strides[0], p.y_st = y_strides[1], p.y_sh = y_strides[2];
        p.lengths = key_lengths;
        p.mask = key_mask;
        p.mask_sb = static_cast<long long>(key_mask_ld);
        p.page_size = 1;
        p.batch = static_cast<int>(batch);
        p.tokens = static_cast<int>(queries);
        p.kv_heads = static_cast<int>(kv_heads);
        p.group = static_cast<int>(group);
        p.size = static_cast<int>(size);
        p.keys = static_cast<int>(keys);
        p.ctas = std::min(dev.num_sms, kB200Sms);
        p.least = kDecodeLeast;
        p.c = c;
        p.parts = workspace_parts(workspace);
        p.status = dev.status;
        return decode_any(p, bf16, s);
    }
    const bool inject = (tuning_bits() & 0x10000000u) != 0 && items == 1;
    const long long wait_limit = inject ? (1ll << 21) : (1ll << 32);
    const bool single = keys <= kTileKeys;
    const unsigned key_rows = single ? static_cast<unsigned>((keys + 15) / 16 * 16) : kTileKeys;
    CUtensorMap mq, mk, mv, my;
    rc = encode_heads(dev, &mq, q, size, queries, heads, batch, q_strides[1], q_strides[2], q_strides[0], 128);
    if (rc == kSuccess) rc = encode_heads(dev, &mk, k, size, keys, kv_heads, batch, k_strides[1], k_strides[2], k_strides[0], key_rows);
    if (rc == kSuccess) rc = encode_heads(dev, &mv, v, size, keys, kv_heads, batch, v_strides[1], v_strides[2], v_strides[0], key_rows);
    if (rc == kSuccess) rc = encode_heads(dev, &my, y, size, queries, heads, batch, y_strides[1], y_strides[2], y_strides[0], 32, !single && size <= 64 ? 32 : 64);
    if (rc != kSuccess) return rc;
    if (single) {
        const long long q_tiles = static_cast<long long>((queries + 127) / 128), tiles = q_tiles * static_cast<long long>(heads) * static_cast<long long>(batch);
        if (tiles > INT_MAX) return kInvalidDimension;
        ShortParams p{};
        p.batch = static_cast<int>(batch);
        p.queries = static_cast<int>(queries);
        p.keys = static_cast<int>(keys);
        p.heads = static_cast<int>(heads);
        p.group = static_cast<int>(group);
        p.size = static_cast<int>(size);
        p.lengths = key_lengths;
        p.mask = key_mask;
        p.mask_sb = static_cast<long long>(key_mask_ld);
        p.q_tiles = static_cast<int>(q_tiles);
        p.tiles = static_cast<int>(tiles);
        p.key_rows = static_cast<int>(key_rows);
        p.k_batched = k_strides[0] != 0;
        p.v_batched = v_strides[0] != 0;
        p.q_batched = q_strides[0] != 0;
        p.c = c;
        p.y = static_cast<char*>(y);
        p.y_sb = y_strides[0], p.y_st = y_strides[1], p.y_sh = y_strides[2];
        p.status = dev.status;
        p.wait_limit = wait_limit;
        p.withhold = inject ? 1 : 0;
        if (size <= 64) return bf16 ? short_launch<true, 64>(p, dev.num_sms, mq, mk, mv, my, s) : short_launch<false, 64>(p, dev.num_sms, mq, mk, mv, my, s);
        return bf16 ? short_launch<true, 128>(p, dev.num_sms, mq, mk, mv, my, s) : short_launch<false, 128>(p, dev.num_sms, mq, mk, mv, my, s);
    }
    TilesParams p{};
    p.batch = static_cast<int>(batch);
    p.queries = static_cast<int>(queries);
    p.keys = static_cast<int>(keys);
    p.heads = static_cast<int>(heads);
    p.group = static_cast<int>(group);
    p.size = static_cast<int>(size);
    p.lengths = key_lengths;
    p.mask = key_mask;
    p.mask_sb = static_cast<long long>(key_mask_ld);
    p.q_pairs = static_cast<int>((queries + 255) / 256);
    const long long units = items * static_cast<long long>((keys + kTileKeys - 1) / kTileKeys);
    p.ctas = static_cast<int>(std::min<long long>(units, std::min(dev.num_sms, kB200Sms)));
    p.y = static_cast<char*>(y);
    p.y_sb = y_strides[0], p.y_st = y_strides[1], p.y_sh = y_strides[2];
    p.parts = workspace_parts(workspace);
    p.q_batched = q_strides[0] != 0;
    p.k_batched = k_strides[0] != 0;
    p.v_batched = v_strides[0] != 0;
    p.c = c;
    p.status = dev.status;
    p.wait_limit = wait_limit;
    p.withhold = inject ? 1 : 0;
    if (size <= 64) return bf16 ? tiles_launch<true, 64>(p, mq, mk, mv, my, s) : tiles_launch<false, 64>(p, mq, mk, mv, my, s);
    return bf16 ? tiles_launch<true, 128>(p, mq, mk, mv, my, s) : tiles_launch<false, 128>(p, mq, mk, mv, my, s);
}

size_t dlf_b200_paged_attention_workspace_bytes(size_t batch, size_t heads, size_t kv_heads, size_t size) {
    (void)batch;
    (void)heads;
    (void)kv_heads;
    return decode_workspace(size);
}

int dlf_b200_paged_attention(const dlf_b200_paged_attention_args* args, void* workspace, size_t workspace_bytes, void* stream) {
    if (args == nullptr) return kInvalidValue;
    const auto& [dtype, scale, batch, heads, kv_heads, size, num_pages, page_size, table_width, table_ld, q_strides, k_strides, v_strides, y_strides,
                 q, k_pages, v_pages, y, page_table, lengths] = *args;
    int rc = head_args(dtype, heads, kv_heads, size);
    if (rc != kSuccess) return rc;
    if (batch == 0 || num_pages == 0 || page_size == 0 || table_width == 0 || batch > 65535 || num_pages > INT_MAX || page_size > INT_MAX ||
        static_cast<double>(table_width) * static_cast<double>(page_size) > INT_MAX / 2)
        return kInvalidDimension;
    if (!scale_ok(scale)) return kInvalidValue;
    if (q == nullptr) return kInvalidMatrixA;
    if (k_pages == nullptr || v_pages == nullptr || page_table == nullptr || lengths == nullptr)
        return kInvalidMatrixB;
    if (y == nullptr) return kInvalidMatrixC;
    if (table_ld < table_width && batch > 1) return kInvalidLeadDimB;
    if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(y) ||
        !strides_ok({q_strides[0], q_strides[1], k_strides[0], k_strides[1], k_strides[2], v_strides[0], v_strides[1], v_strides[2], y_strides[0],
                     y_strides[1]}))
        return kNotImplemented;
    if ((batch > 1 && y_strides[0] == 0) || (heads > 1 && y_strides[1] == 0)) return kInvalidLeadDimC;
    if (static_cast<double>(batch) * heads * (static_cast<double>(table_width) * page_size / kDecodeUnit + 1.0) > 2147483647.0) return kInvalidDimension;
    if (workspace == nullptr || workspace_bytes < dlf_b200_paged_attention_workspace_bytes(batch, heads, kv_heads, size)) return kInsufficientMemoryTemp;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    StreamDevice guard(s);
    if (guard.rc != kSuccess) return guard.rc;
    OperatorDevice dev;
    rc = operator_device(&dev);
    if (rc != kSuccess) return rc;
    rc = attention_device(dev);
    if (rc != kSuccess) return rc;
    clear_stale_error();
    DecodeParams p{};
    p.q = static_cast<const char*>(q);
    p.k = static_cast<const char*>(k_pages);
    p.v = static_cast<const char*>(v_pages);
    p.y = static_cast<char*>(y);
    p.q_sb = q_strides[0], p.q_sh = q_strides[1];
    p.k_sb = k_strides[0], p.k_st = k_strides[1], p.k_sh = k_strides[2];
    p.v_sb = v_strides[0], p.v_st = v_strides[1], p.v_sh = v_strides[2];
    p.y_sb = y_strides[0], p.y_sh = y_strides[1];
    p.lengths = lengths;
    p.table = page_table;
    p.table_sb = static_cast<long long>(table_ld);
    p.page_size = static_cast<int>(page_size);
    p.num_pages = static_cast<int>(num_pages);
    p.batch = static_cast<int>(batch);
    p.tokens = 1;
    p.kv_heads = static_cast<int>(kv_heads);
    p.group = static_cast<int>(heads / kv_heads);
    p.size = static_cast<int>(size);
    p.keys = static_cast<int>(table_width * page_size);
    p.ctas = std::min(dev.num_sms, kB200Sms);
    p.least = kDecodeLeast;
    p.c = scale * kLog2e;
    p.parts = workspace_parts(workspace);
    p.status = dev.status;
    return decode_any(p, dtype == DLF_B200_BFLOAT16, s);
}

int dlf_b200_paged_append(const dlf_b200_paged_append_args* args, void* stream) {
    if (args == nullptr) return kInvalidValue;
    const auto& [dtype, tokens, kv_heads, size, batch, num_pages, page_size, table_width, table_ld, k_strides, v_strides, kp_strides, vp_strides, k, v,
                 k_pages, v_pages, page_table, positions, sequences] = *args;
    int rc = head_args(dtype, kv_heads, kv_heads, size);
    if (rc != kSuccess) return rc;
    if (tokens == 0 || batch == 0 || num_pages == 0 || page_size == 0 || table_width == 0 || tokens > INT_MAX || batch > INT_MAX || num_pages > INT_MAX ||
        page_size > INT_MAX || table_width > INT_MAX || kv_heads * size > INT_MAX)
        return kInvalidDimension;
    if (sequences == nullptr && tokens > batch) return kInvalidDimension;
    if (k == nullptr || v == nullptr) return kInvalidMatrixA;
    if (page_table == nullptr || positions == nullptr) return kInvalidMatrixB;
    if (k_pages == nullptr || v_pages == nullptr) return kInvalidMatrixC;
    if (table_ld < table_width && batch > 1) return kInvalidLeadDimB;
    if (!aligned16(k) || !aligned16(v) || !aligned16(k_pages) || !aligned16(v_pages) ||
        !strides_ok({k_strides[0], k_strides[1], v_strides[0], v_strides[1], kp_strides[0], kp_strides[1], kp_strides[2], vp_strides[0], vp_strides[1],
                     vp_strides[2]}))
        return kNotImplemented;
    for (const size_t* st : {&kp_strides[0], &vp_strides[0]})  // (a place of its own for every token and head)
        if ((num_pages > 1 && st[0] == 0) || (page_size > 1 && st[1] == 0) || (kv_heads > 1 && st[2] == 0)) return kInvalidLeadDimC;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    StreamDevice guard(s);
    if (guard.rc != kSuccess) return guard.rc;
    OperatorDevice dev;
    rc = operator_device(&dev);
    if (rc != kSuccess) return rc;
    clear_stale_error();
    AppendParams p{};
    p.k = static_cast<const char*>(k);
    p.v = static_cast<const char*>(v);
    p.k_pages = static_cast<char*>(k_pages);
    p.v_pages = static_cast<char*>(v_pages);
    p.k_st = k_strides[0], p.k_sh = k_strides[1], p.v_st = v_strides[0], p.v_sh = v_strides[1];
    p.kp_sb = kp_strides[0], p.kp_st = kp_strides[1], p.kp_sh = kp_strides[2];
    p.vp_sb = vp_strides[0], p.vp_st = vp_strides[1], p.vp_sh = vp_strides[2];
    p.table = page_table;
    p.table_sb = static_cast<long long>(table_ld);
    p.positions = positions;
    p.sequences = sequences;
    p.tokens = static_cast<int>(tokens);
    p.batch = static_cast<int>(batch);
    p.table_width = static_cast<int>(std::min<size_t>(table_width, INT_MAX / 2));
    p.page_size = static_cast<int>(page_size);
    p.num_pages = static_cast<int>(num_pages);
    p.kv_heads = static_cast<int>(kv_heads);
    p.size = static_cast<int>(size);
    p.status = dev.status;
    const long long total = static_cast<long long>(tokens) * static_cast<long long>(kv_heads) * (static_cast<long long>(size) / 8);
    CUDA_TRY(launch_dependent(paged_append_kernel, static_cast<unsigned>(std::min<long long>((total + 255) / 256, 16ll * dev.num_sms)), 256u, 0, s, p));
    count_launch();
    CUDA_TRY(cudaGetLastError());
    return kSuccess;
}

}  // extern "C"
