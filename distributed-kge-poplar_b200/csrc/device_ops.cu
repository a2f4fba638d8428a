// The operators of a softmax over all candidates on device arrays: checks of their arguments and their launches.
#include "device_ops.hpp"

#include <cuda.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "adamw.cuh"
#include "log_probs.cuh"
#include "rows8.cuh"

namespace kge {
namespace {

void need(bool ok, const char* what) {
    if (!ok) fail(KGE_INVALID_ARGUMENT, what);
}
bool aligned_to(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
size_t type_bytes(int type, const char* what) {
    if (type != KGE_F32 && type != KGE_F16 && type != KGE_BF16) fail(KGE_INVALID_ARGUMENT, msg() << what << ": the element type must be KGE_F32, KGE_F16 or KGE_BF16, not " << type);
    return type == KGE_F32 ? 4 : 2;
}
// fn(T()) for the element type named.
template <class Fn>
void with_type(int type, Fn&& fn) {
    if (type == KGE_F32) fn(float());
    else if (type == KGE_F16) fn(__half());
    else fn(__nv_bfloat16());
}
unsigned grid_of(size_t blocks, const char* what) {
    if (blocks > 0x7fffffffu) fail(KGE_INVALID_ARGUMENT, msg() << what << ": too large for one launch");
    return (unsigned)blocks;
}
// Allows a kernel its dynamic shared memory, once per device.
template <auto Kernel>
void allow_shared_memory(size_t bytes) {
    static std::atomic<uint64_t> done{0};
    const int slot = current_device_slot();
    if (slot >= 0 && (done.load() >> slot & 1)) return;
    KGE_CUDA(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    if (slot >= 0) done.fetch_or((uint64_t)1 << slot);
}

constexpr size_t kMostColumns = 0x7fffffffu - 65536;  // a column and a vector past it fit an int

lp::Scores checked_scores(const kge_scores& s, const char* what) {
    const size_t bytes = type_bytes(s.float_type, what);
    if (s.cols > kMostColumns) fail(KGE_INVALID_ARGUMENT, msg() << what << ": " << s.cols << " columns, " << kMostColumns << " are the most");
    if (s.rows > 1 && s.row_stride < (long long)s.cols) fail(KGE_INVALID_ARGUMENT, msg() << what << ": rows of " << s.cols << " columns, " << s.row_stride << " apart");
    if (!(s.scale > 0.f) || !std::isfinite(s.scale * lp::kLog2e)) fail(KGE_INVALID_ARGUMENT, msg() << what << ": scale must be positive and finite, not " << s.scale);
    if (s.rows && s.cols && !s.x) fail(KGE_INVALID_ARGUMENT, msg() << what << ": null scores");
    if (!aligned_to(s.x, bytes)) fail(KGE_INVALID_ARGUMENT, msg() << what << ": scores are not aligned to their type");
    if (s.mask && s.mask_stride != 0 && s.rows > 1 && s.mask_stride < (long long)s.cols)
        fail(KGE_INVALID_ARGUMENT, msg() << what << ": mask rows of " << s.cols << " columns, " << s.mask_stride << " apart");
    return lp::Scores{s.x, s.mask, s.count, s.target, s.row_stride, s.mask_stride, (int)s.cols, s.scale * lp::kLog2e, s.scale};
}

}  // namespace

// ---------------------------------------------------------------------------

namespace {

// A row is one block's.  Each kernel holds 64 registers a thread, 1024 threads to an SM, and blocks are as large as leaves all rows at work
// at once: 1024 threads for a row an SM, 512 for two.  A row more than that waits for a second, nearly empty wave, and smaller blocks are
// sooner done: of 20 001 bf16 scores 148 rows 6.7 us by blocks of 1024; 149 11.5, by 512 5.4; with lists of 100 13.1; 21.1, by 512
// 11.5; 297 rows by 512 8.2, by 256 7.9; of 100 003 bf16 scores with lists of 100 148 rows 18.0 by 1024; 149 30.5, by 512 20.4.
// (128 rows of those in parts of 256 threads, with a second kernel to join them: 31.0, as rows of one block each 17.7.)
// Rows are cut into parts, four to an SM, where there are too few of them for that (4 rows of 2 500 001 fp32 scores 12.1 us, by one block a
// row 162; 60 of 200 001 bf16 ones 11.1, 16.2) or the groups of vectors of their lists do not fit a block's shared memory; two to an SM with
// lists, which each part makes (4 rows with lists of 100 28.5, with four to an SM 30.3).  Many short rows go to blocks of 128 threads, whose
// sums are joined sooner: 4096 rows of 10 001 bf16 scores 23.6 us, by blocks of 256 31.0, with lists of 10 39.3 and 60.6; 4096 of
// 20 001 fp32 ones, 5001 vectors each, take 59.6 us either way.
struct LogProbsPlan {
    int threads, parts, vectors;
    size_t sums_bytes, bytes;
};
LogProbsPlan log_probs_plan(size_t rows, size_t cols, size_t n_best, size_t width) {
    LogProbsPlan p;
    const size_t all = (cols + 2 * width - 2) / width;  // whatever a row's first vector leaves out
    const auto most = [](int threads) {
        const int groups = threads == 1024 ? lp::Lists<1024>::kGroups : threads == 512 ? lp::Lists<512>::kGroups : threads == 256 ? lp::Lists<256>::kGroups : lp::Lists<128>::kGroups;
        return (size_t)threads * groups * lp::kGroup;
    };
    size_t parts = 1;
    if (all <= 512 || (rows >= 4 * kSmCount && all <= (n_best ? most(128) : 4096))) {
        p.threads = 128;
    } else {
        p.threads = rows <= kSmCount ? 1024 : rows <= 2 * kSmCount ? 512 : 256;
        while (p.threads > 256 && (size_t)p.threads * 2 > all) p.threads /= 2;  // two vectors a thread at least
        if ((n_best && all > most(p.threads)) || (rows <= kSmCount / 2 && (all > 16384 || (rows <= 16 && all >= 2048)))) {
            p.threads = 256;
            parts = std::max((all + most(256) - 1) / most(256), std::min((n_best ? 2 : 4) * kSmCount / std::max<size_t>(1, rows), all / 1024));
        }
    }
    p.vectors = (int)std::max<size_t>(1, (all + parts - 1) / parts);
    p.parts = (int)std::max<size_t>(1, (all + p.vectors - 1) / p.vectors);
    p.sums_bytes = round_up(rows * (size_t)p.parts * sizeof(float4), 256);
    p.bytes = p.parts > 1 ? p.sums_bytes + rows * (size_t)p.parts * n_best * sizeof(unsigned long long) : 0;
    return p;
}

template <class T>
void launch_log_probs(int threads, unsigned blocks, const lp::Scores& s, const lp::Out& o, const lp::Parts& parts, cudaStream_t stream) {
    cudaError_t err;
    if (threads == 128) err = launch_dependent(lp::k_log_probs<T, 128>, dim3(blocks), dim3(128), 0, stream, s, o, parts);
    else if (threads == 256) err = launch_dependent(lp::k_log_probs<T, 256>, dim3(blocks), dim3(256), 0, stream, s, o, parts);
    else if (threads == 512) err = launch_dependent(lp::k_log_probs<T, 512>, dim3(blocks), dim3(512), 0, stream, s, o, parts);
    else err = launch_dependent(lp::k_log_probs<T, 1024>, dim3(blocks), dim3(1024), 0, stream, s, o, parts);
    KGE_CUDA(err);
}

}  // namespace

size_t log_probs_workspace(size_t rows, size_t cols, size_t n_best) {
    if (rows == 0 || cols > kMostColumns || n_best > (size_t)lp::kMaxBest) return 0;
    return std::max(log_probs_plan(rows, cols, n_best, 4).bytes, log_probs_plan(rows, cols, n_best, 8).bytes);
}

void log_probs(const kge_scores& scores, const kge_log_probs_out& out, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
    const char* const what = "kge_op_log_probs";
    const lp::Scores s = checked_scores(scores, what);
    if (out.n_best > (size_t)lp::kMaxBest) fail(KGE_INVALID_ARGUMENT, msg() << what << ": n_best is " << out.n_best << ", " << lp::kMaxBest << " is the most");
    if (scores.rows == 0) return;
    need(out.log_prob && out.entropy && out.log_sum && out.row_state && (!out.n_best || (out.best_log_prob && out.best_index)), "kge_op_log_probs: null output");
    need(aligned_to(out.row_state, 16), "kge_op_log_probs: row_state is not aligned to 16 bytes");
    const size_t wanted = log_probs_workspace(scores.rows, scores.cols, out.n_best);
    if (wanted) {
        if (workspace_bytes < wanted || !workspace) fail(KGE_INVALID_ARGUMENT, msg() << what << ": a workspace of " << wanted << " bytes is wanted, not " << workspace_bytes);
        need(aligned_to(workspace, 256), "kge_op_log_probs: the workspace is not aligned to 256 bytes");
    }
    const LogProbsPlan p = log_probs_plan(scores.rows, scores.cols, out.n_best, 16 / type_bytes(scores.float_type, what));
    const lp::Out o{out.log_prob, out.entropy, out.log_sum, reinterpret_cast<float4*>(out.row_state), out.best_log_prob, out.best_index, (int)out.n_best};
    const lp::Parts parts{p.parts, p.vectors, static_cast<float4*>(workspace),
                          reinterpret_cast<unsigned long long*>(static_cast<char*>(workspace) + (workspace ? p.sums_bytes : 0))};
    const unsigned blocks = grid_of(scores.rows * (size_t)p.parts, what);
    with_type(scores.float_type, [&](auto t) {
        using T = decltype(t);
        launch_log_probs<T>(p.threads, blocks, s, o, parts, stream);
        // a short join has few lists to look through, a long one is done sooner by more warps
        if (p.parts > 32 && out.n_best) {
            const cudaError_t err = launch_dependent(lp::k_join_parts<T, 1024>, dim3((unsigned)scores.rows), dim3(1024), 0, stream, s, o, parts);
            KGE_CUDA(err);
        } else if (p.parts > 1) {
            const cudaError_t err = launch_dependent(lp::k_join_parts<T, 256>, dim3((unsigned)scores.rows), dim3(256), 0, stream, s, o, parts);
            KGE_CUDA(err);
        }
    });
}

void log_probs_grad(const kge_scores& scores, const float* row_state, const float* grad_log_prob, const float* grad_entropy, size_t n_best,
                    const int32_t* best_index, const float* grad_best, void* grad_x, long long grad_row_stride, cudaStream_t stream) {
    const char* const what = "kge_op_log_probs_grad";
    const lp::Scores s = checked_scores(scores, what);
    if (n_best > (size_t)lp::kMaxBest) fail(KGE_INVALID_ARGUMENT, msg() << what << ": n_best is " << n_best << ", " << lp::kMaxBest << " is the most");
    if (scores.rows == 0 || scores.cols == 0) return;
    need(row_state && grad_x, "kge_op_log_probs_grad: null argument");
    need(aligned_to(row_state, 16), "kge_op_log_probs_grad: row_state is not aligned to 16 bytes");
    need(aligned_to(grad_x, type_bytes(scores.float_type, what)), "kge_op_log_probs_grad: the gradient is not aligned to its type");
    need(!grad_best || !n_best || best_index, "kge_op_log_probs_grad: alternatives with a gradient but no indices");
    if (scores.rows > 1 && grad_row_stride < (long long)scores.cols)
        fail(KGE_INVALID_ARGUMENT, msg() << what << ": gradient rows of " << scores.cols << " columns, " << grad_row_stride << " apart");
    need(grad_x != scores.x || scores.rows == 1 || grad_row_stride == scores.row_stride, "kge_op_log_probs_grad: a gradient in the scores' place has their row stride");
    const size_t width = 16 / type_bytes(scores.float_type, what);
    const size_t per_block = (size_t)lp::kGradThreads * lp::kGroup;
    const size_t blocks = ((scores.cols + 2 * width - 2) / width + per_block - 1) / per_block;  // whatever a row's first vector leaves out
    const lp::GradArgs g{reinterpret_cast<const float4*>(row_state), grad_log_prob, grad_entropy, best_index, n_best ? grad_best : nullptr,
                         grad_x, grad_row_stride, (int)n_best, (int)blocks, (uint32_t)scores.rows};
    const unsigned grid = grid_of(scores.rows * blocks, what);
    with_type(scores.float_type, [&](auto t) { KGE_CUDA(launch_dependent(lp::k_log_probs_grad<decltype(t)>, dim3(grid), dim3(lp::kGradThreads), 0, stream, s, g)); });
}

// ---------------------------------------------------------------------------

void rows8_bytes(size_t rows, size_t cols, size_t* values, size_t* exponents) {
    *values = rows * rows8::value_stride(cols);
    *exponents = (rows + 127) / 128 * rows8::groups_of(cols) * rows8::kGroupBytes;
}

void quantise_rows(const void* x, int float_type, size_t rows, size_t cols, long long row_stride, bool transposed, uint8_t* values,
                   uint8_t* exponents, cudaStream_t stream) {
    const char* const what = "kge_op_quantise_rows";
    const size_t bytes = type_bytes(float_type, what);
    if (rows > 1 && row_stride < (long long)cols) fail(KGE_INVALID_ARGUMENT, msg() << what << ": rows of " << cols << " columns, " << row_stride << " apart");
    if (rows == 0 || cols == 0) return;
    need(x && values && exponents, "kge_op_quantise_rows: null argument");
    need(aligned_to(x, bytes), "kge_op_quantise_rows: x is not aligned to its type");
    need(aligned_to(values, 16) && aligned_to(exponents, 16), "kge_op_quantise_rows: values and exponents must be aligned to 16 bytes");
    with_type(float_type, [&](auto t) {
        using T = decltype(t);
        const T* const src = static_cast<const T*>(x);
        if (!transposed) {
            const size_t blocks = rows8::blocks_of(cols), units = round_up(rows, 128) * blocks, per = 8 * 4;
            if (units > 0xffffff00u) fail(KGE_INVALID_ARGUMENT, msg() << what << ": " << rows << " x " << cols << " is too large for one launch");
            const cudaError_t err = launch_dependent(rows8::k_quantise_rows<T>, dim3((unsigned)((units + per - 1) / per)), dim3(256), 0, stream, src, (uint32_t)rows, cols,
                                                     row_stride, (uint32_t)blocks, (uint32_t)rows8::groups_of(cols), (uint32_t)units, values, exponents);
            KGE_CUDA(err);
        } else {
            const size_t groups = rows8::groups_of(rows), tiles = round_up(cols, 128) / rows8::kTurnCols;
            const cudaError_t err = launch_dependent(rows8::k_quantise_columns<T>, dim3(grid_of(tiles * groups * 4, what)), dim3(256), 0, stream, src, rows, cols, row_stride,
                                                     groups, values, exponents);
            KGE_CUDA(err);
        }
    });
}

namespace {

// Sizes whose plan is counted in ints: others are refused, and want no workspace.
bool product_fits(size_t m, size_t n, size_t k) { return m <= 0x7fffffffu && n <= 0x7fffffffu - 65536 && k <= 0x7fffffffu - 65536; }

struct ProductPlan {
    int tile_m, m_tiles, n_tiles, blocks, splits, chunk;
};
ProductPlan product_plan(size_t m, size_t n, size_t k) {
    ProductPlan p;
    p.n_tiles = (int)((n + rows8::kTileN - 1) / rows8::kTileN);
    p.tile_m = m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : m <= 128 ? 128 : 256;
    // Blocks that keep their queries have a tile's 128 (512 x 500 000 x 256: 117 us, with 256, whose accumulators share columns, 148);
    // where the sum has to be split, smaller tiles need half the parts and so half the partial sums.
    if (p.tile_m == 256 && rows8::blocks_of(k) <= (size_t)rows8::Tile<128, true>::kMostResident && m <= (size_t)kSmCount * 128) p.tile_m = 128;
    if (p.tile_m == 256 && (long long)((m + 255) / 256) * p.n_tiles < kSmCount / 2) p.tile_m = 128;
    p.m_tiles = (int)((m + p.tile_m - 1) / p.tile_m);
    p.chunk = (int)std::min<size_t>(p.n_tiles, std::max<size_t>(16, ((size_t)32 << 20) / (rows8::kTileN * rows8::value_stride(std::max<size_t>(k, 1)))));
    p.blocks = (int)rows8::blocks_of(k);
    const long long tiles = (long long)p.m_tiles * p.n_tiles;
    p.splits = (int)std::max<long long>(1, std::min<long long>(tiles ? kSmCount / tiles : 1, p.blocks / 4));
    return p;
}

CUtensorMap encoded_map(CUtensorMapDataType type, const void* base, cuuint64_t cols, cuuint64_t rows, cuuint64_t stride_bytes, cuuint32_t box_cols, cuuint32_t box_rows,
                        CUtensorMapSwizzle swizzle) {
    tc::EncodeTiledFn encode = tc::encode_tiled_fn();
    if (!encode) fail(KGE_RUNTIME_ERROR, "kge_op_product8: the driver has no cuTensorMapEncodeTiled");
    CUtensorMap map;
    const cuuint64_t dims[2] = {cols, rows}, strides[1] = {stride_bytes};
    const cuuint32_t box[2] = {box_cols, box_rows}, step[2] = {1, 1};
    if (encode(&map, type, 2, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        fail(KGE_RUNTIME_ERROR, "kge_op_product8: a tensor map was refused");
    return map;
}
CUtensorMap rows_map(const uint8_t* values, size_t rows, size_t cols, int box_rows) {
    return encoded_map(CU_TENSOR_MAP_DATA_TYPE_UINT8, values, cols, rows, rows8::value_stride(cols), rows8::kBlock, (cuuint32_t)box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}
template <class T>
constexpr CUtensorMapDataType map_type() {
    return sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

template <int TM, class TOut, bool RESIDENT>
void launch_product(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& out, const rows8::ProductArgs& g, int grid, cudaStream_t stream) {
    using L = rows8::Tile<TM, RESIDENT>;
    allow_shared_memory<rows8::k_product8<TM, TOut, RESIDENT>>(L::smem());
    const cudaError_t err = launch_dependent(rows8::k_product8<TM, TOut, RESIDENT>, dim3(grid), dim3(L::kThreads), L::smem(), stream, a, b, out, g);
    KGE_CUDA(err);
}
template <int TM, class TOut>
void launch_product(const CUtensorMap& a, const CUtensorMap& b, rows8::ProductArgs g, cudaStream_t stream) {
    if constexpr (TM <= 128) {
        using Kept = rows8::Tile<TM, true>;
        if (g.blocks <= Kept::kMostResident && g.splits == 1 && g.m_tiles <= kSmCount) {
            CUtensorMap out = b;  // where results are stored directly, any map
            g.stages = Kept::lone_stages(g.blocks);
            // A box that ends inside 16 bytes of a row is written to their end, past the row's columns: where the rows' width is no multiple
            // of 16 bytes the last tile is stored directly.
            if (TM >= 64 && aligned_to(g.out, 16) && (g.m == 1 || g.out_stride * (long long)sizeof(TOut) % 16 == 0))
                g.boxes = (size_t)g.n * sizeof(TOut) % 16 == 0 ? g.n_tiles : g.n / rows8::kTileN;
            if (g.boxes)
                out = encoded_map(map_type<TOut>(), g.out, (cuuint64_t)g.n, (cuuint64_t)g.m, round_up((size_t)std::max<long long>(g.out_stride, g.n) * sizeof(TOut), 16),
                                  rows8::kBoxColumns<TOut>, rows8::kBoxRows<TOut>, sizeof(TOut) == 4 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B);
            launch_product<TM, TOut, true>(a, b, out, g, std::min(g.n_tiles, kSmCount / g.m_tiles) * g.m_tiles, stream);
            return;
        }
    }
    g.stages = rows8::Tile<TM, false>::kPairStages;
    launch_product<TM, TOut, false>(a, b, b, g, std::min(g.n_tiles * g.m_tiles * g.splits, kSmCount), stream);
}
template <class TOut>
void launch_product(int tile_m, const CUtensorMap& a, const CUtensorMap& b, const rows8::ProductArgs& g, cudaStream_t stream) {
    if (tile_m == 16) launch_product<16, TOut>(a, b, g, stream);
    else if (tile_m == 32) launch_product<32, TOut>(a, b, g, stream);
    else if (tile_m == 64) launch_product<64, TOut>(a, b, g, stream);
    else if (tile_m == 128) launch_product<128, TOut>(a, b, g, stream);
    else launch_product<256, TOut>(a, b, g, stream);
}

}  // namespace

size_t product8_workspace(size_t m, size_t n, size_t k) {
    if (m == 0 || n == 0 || k == 0 || !product_fits(m, n, k)) return 0;
    const ProductPlan p = product_plan(m, n, k);
    return p.splits > 1 ? (size_t)p.splits * m * n * sizeof(float) : 0;
}

void product8(const uint8_t* a_values, const uint8_t* a_exponents, size_t m, const uint8_t* b_values, const uint8_t* b_exponents, size_t n,
              size_t k, void* out, int out_type, long long out_row_stride, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
    const char* const what = "kge_op_product8";
    const size_t bytes = type_bytes(out_type, what);
    if (!product_fits(m, n, k)) fail(KGE_INVALID_ARGUMENT, msg() << what << ": " << m << " x " << n << " x " << k << " is too large");
    if (m > 1 && out_row_stride < (long long)n) fail(KGE_INVALID_ARGUMENT, msg() << what << ": rows of " << n << " results, " << out_row_stride << " apart");
    if (m == 0 || n == 0) return;
    need(out, "kge_op_product8: null output");
    need(aligned_to(out, bytes), "kge_op_product8: the output is not aligned to its type");
    if (k == 0) {
        KGE_CUDA(cudaMemset2DAsync(out, (size_t)std::max<long long>(out_row_stride, (long long)n) * bytes, 0, n * bytes, m, stream));
        return;
    }
    need(a_values && a_exponents && b_values && b_exponents, "kge_op_product8: null operand");
    need(aligned_to(a_values, 16) && aligned_to(a_exponents, 16) && aligned_to(b_values, 16) && aligned_to(b_exponents, 16),
         "kge_op_product8: operands must be aligned to 16 bytes");
    const ProductPlan p = product_plan(m, n, k);
    if ((long long)p.m_tiles * p.n_tiles * p.splits > 0x7fffffff) fail(KGE_INVALID_ARGUMENT, msg() << what << ": " << m << " x " << n << " is too large");
    const size_t wanted = product8_workspace(m, n, k);
    if (wanted) {
        if (workspace_bytes < wanted || !workspace) fail(KGE_INVALID_ARGUMENT, msg() << what << ": a workspace of " << wanted << " bytes is wanted, not " << workspace_bytes);
        need(aligned_to(workspace, 256), "kge_op_product8: the workspace is not aligned to 256 bytes");
    }
    const CUtensorMap a = rows_map(a_values, m, k, p.tile_m), b = rows_map(b_values, n, k, rows8::kTileN);
    rows8::ProductArgs g{a_exponents, b_exponents, out, out_row_stride, 0, (int)m, (int)n, p.blocks, (p.blocks + 3) / 4, p.n_tiles, p.m_tiles, p.splits, p.chunk, 0, 0};
    if (p.splits > 1) {
        g.out = workspace;
        g.out_stride = (long long)n;
        g.split_stride = (long long)m * (long long)n;
        launch_product<float>(p.tile_m, a, b, g, stream);
        with_type(out_type, [&](auto t) {
            using T = decltype(t);
            const cudaError_t err = launch_dependent(rows8::k_add_splits<T>, dim3(grid_of((m * n + 255) / 256, what)), dim3(256), 0, stream, static_cast<const float*>(workspace),
                                                     g.split_stride, p.splits, (int)m, (int)n, static_cast<T*>(out), out_row_stride);
            KGE_CUDA(err);
        });
    } else {
        with_type(out_type, [&](auto t) { launch_product<decltype(t)>(p.tile_m, a, b, g, stream); });
    }
    KGE_CUDA(cudaGetLastError());
}

bool product8_gave_up() {
    unsigned status = 0;
    KGE_CUDA(cudaDeviceSynchronize());  // the copy alone would not wait for streams that do not wait for the default stream
    KGE_CUDA(cudaMemcpyFromSymbol(&status, rows8::g_product8_status, sizeof status));
    if (status) {
        const unsigned zero = 0;
        KGE_CUDA(cudaMemcpyToSymbol(rows8::g_product8_status, &zero, sizeof zero));
    }
    return status != 0;
}

// ---------------------------------------------------------------------------

namespace {

template <class TP, class TG, int MAX>
void launch_adamw(const adamw::Table<adamw::kMaxTensors>& all, const adamw::Params& p, const kge_adamw_args& a, cudaStream_t stream) {
    adamw::Table<MAX> table;
    table.n = all.n;
    std::copy(all.t, all.t + all.n, table.t);
    const uint32_t per = adamw::kThreads / 32 * (a.state_bits == 8 ? 1 : adamw::kBlocksPerWarp), grid = (all.t[all.n - 1].units_end + per - 1) / per;
    cudaError_t err;
    if (a.state_bits == 8)
        err = launch_dependent(adamw::k_adamw8<TP, TG, MAX>, dim3(grid), dim3(adamw::kThreads), 0, stream, table, p, static_cast<uint8_t*>(a.adam_m),
                               static_cast<uint8_t*>(a.adam_v), a.m_exponent, a.v_exponent);
    else
        err = launch_dependent(adamw::k_adamw32<TP, TG, MAX>, dim3(grid), dim3(adamw::kThreads), 0, stream, table, p, static_cast<float*>(a.adam_m), static_cast<float*>(a.adam_v));
    KGE_CUDA(err);
}
template <class TP, class TG>
void launch_adamw(const adamw::Table<adamw::kMaxTensors>& all, const adamw::Params& p, const kge_adamw_args& a, cudaStream_t stream) {
    // few tensors take a table of their own size along with the launch: a call with one 4.8 us, with six 5.2, in the large table's 10 KB 5.3
    // and 5.6; captured steps do not see it
    if (all.n <= 16) launch_adamw<TP, TG, 16>(all, p, a, stream);
    else launch_adamw<TP, TG, adamw::kMaxTensors>(all, p, a, stream);
}

}  // namespace

void adamw_step(const kge_adamw_args& a, const kge_adamw_tensor* tensors, size_t n_tensors, cudaStream_t stream) {
    const char* const what = "kge_op_adamw";
    if (a.param_type != KGE_F32 && a.param_type != KGE_BF16) fail(KGE_INVALID_ARGUMENT, msg() << what << ": parameters must be KGE_F32 or KGE_BF16, not " << a.param_type);
    const size_t param_bytes = a.param_type == KGE_F32 ? 4 : 2, grad_bytes = type_bytes(a.grad_type, what);
    if (a.state_bits != 8 && a.state_bits != 32) fail(KGE_INVALID_ARGUMENT, msg() << what << ": state_bits must be 8 or 32, not " << a.state_bits);
    // (float)epsilon must be a normal number: 0 makes 0 / 0 of values that have had no gradient yet
    if (!((float)a.epsilon >= FLT_MIN && (float)a.epsilon <= FLT_MAX)) fail(KGE_INVALID_ARGUMENT, msg() << what << ": epsilon must be a normal fp32 number above 0, not " << a.epsilon);
    // (1 - beta) times the scale, or its square, is one fp32 factor: where that is no normal number the moments would be lost or infinite
    const auto held = [&](double beta, double scale) {
        const float factor = (float)std::fabs((1. - beta) * scale);
        return beta == 1. || scale == 0. || !std::isfinite(a.grad_scale) || (factor >= FLT_MIN && factor <= FLT_MAX);
    };
    if (!held(a.beta_m, a.grad_scale) || !held(a.beta_v, a.grad_scale * a.grad_scale) || (a.grad_scale != 0. && a.grad_scale * a.grad_scale == 0.))
        fail(KGE_INVALID_ARGUMENT, msg() << what << ": grad_scale is " << a.grad_scale << ": (1 - beta) times its square must be a normal fp32 number");
    need(n_tensors == 0 || tensors, "kge_op_adamw: null tensors");
    const adamw::Params p{(float)a.beta_m, (float)((1. - a.beta_m) * a.grad_scale), (float)a.beta_v, (float)((1. - a.beta_v) * a.grad_scale * a.grad_scale), (float)a.epsilon,
                          (float)a.decay, (float)a.step_size, (float)a.inv_sqrt_correction, a.key, a.schedule};
    adamw::Table<adamw::kMaxTensors> table;
    table.n = 0;
    uint32_t units = 0;
    const size_t unit_values = adamw::kBlock * (a.state_bits == 8 ? 4 : 1);
    for (size_t i = 0; i < n_tensors; ++i) {
        const kge_adamw_tensor& t = tensors[i];
        if (!t.size) continue;
        if (!t.param || !t.grad) fail(KGE_INVALID_ARGUMENT, msg() << what << ": tensor " << i << " has no parameter or no gradient");
        if (!aligned_to(t.param, param_bytes) || !aligned_to(t.grad, grad_bytes)) fail(KGE_INVALID_ARGUMENT, msg() << what << ": tensor " << i << " is not aligned to its type");
        if (t.first % adamw::kBlock) fail(KGE_INVALID_ARGUMENT, msg() << what << ": the moments of tensor " << i << " begin at " << t.first << ", no multiple of " << adamw::kBlock);
        if ((t.size + adamw::kBlock - 1) / adamw::kBlock > 0x7fffffffu) fail(KGE_INVALID_ARGUMENT, msg() << what << ": tensor " << i << " has " << t.size << " values, too many");
    }
    bool any = false;
    for (size_t i = 0; i < n_tensors; ++i) any = any || tensors[i].size;
    if (!any) return;
    need(a.adam_m && a.adam_v && (a.state_bits == 32 || (a.m_exponent && a.v_exponent)), "kge_op_adamw: null moments");
    need(aligned_to(a.adam_m, 16) && aligned_to(a.adam_v, 16), "kge_op_adamw: the moments are not aligned to 16 bytes");
    need(!a.schedule || aligned_to(a.schedule, 4), "kge_op_adamw: the schedule is not aligned");
    const auto flush = [&] {
        if (table.n == 0) return;
        with_type(a.grad_type, [&](auto g) {
            using TG = decltype(g);
            if (a.param_type == KGE_F32) launch_adamw<float, TG>(table, p, a, stream);
            else launch_adamw<__nv_bfloat16, TG>(table, p, a, stream);
        });
        table.n = 0;
        units = 0;
    };
    for (size_t i = 0; i < n_tensors; ++i) {
        const kge_adamw_tensor& t = tensors[i];
        if (!t.size) continue;
        const uint32_t more = (uint32_t)((t.size + unit_values - 1) / unit_values);
        if (table.n == adamw::kMaxTensors || more > 0x7fffffffu - units) flush();
        units += more;
        const size_t vector = a.state_bits == 8 ? 16 : 0;  // of 8-bit moments' lanes; else four values
        table.t[table.n++] = adamw::Tensor{t.param, t.grad, t.size, t.first, units,
                                           aligned_to(t.param, std::max(vector, 4 * param_bytes)) && aligned_to(t.grad, std::max(vector, 4 * grad_bytes))};
    }
    flush();
}

uint32_t adamw_key(uint32_t seed, uint32_t step) { return adamw::mix(seed * 0x9E3779B9u + step * 0xBB67AE85u); }

void adamw_moments(const uint8_t* adam_m, const uint8_t* m_exponent, const uint8_t* adam_v, const uint8_t* v_exponent, size_t size, void* m_bf16,
                   void* v_bf16, cudaStream_t stream) {
    const char* const what = "kge_op_adamw_moments";
    if (size % adamw::kBlock) fail(KGE_INVALID_ARGUMENT, msg() << what << ": the size is " << size << ", no multiple of " << adamw::kBlock);
    if (size == 0) return;
    need(adam_m && m_exponent && adam_v && v_exponent && m_bf16 && v_bf16, "kge_op_adamw_moments: null argument");
    need(aligned_to(adam_m, 16) && aligned_to(adam_v, 16) && aligned_to(m_bf16, 16) && aligned_to(v_bf16, 16), "kge_op_adamw_moments: moments must be aligned to 16 bytes");
    const size_t per = adamw::kThreads * 8;
    const cudaError_t err = launch_dependent(adamw::k_moments, dim3(grid_of((size + per - 1) / per, what)), dim3(adamw::kThreads), 0, stream, adam_m, m_exponent, adam_v,
                                             v_exponent, size, static_cast<__nv_bfloat16*>(m_bf16), static_cast<__nv_bfloat16*>(v_bf16));
    KGE_CUDA(err);
}

}  // namespace kge
