// C ABI of the scoring and training operators (declared in include/lffw_fp8.h): argument
// validation, the sm_100 device gate and dispatch to the kernel launchers.
#include "lffw_fp8.h"

#include <cuda_runtime_api.h>

#include <cmath>

#include "launch.h"

namespace {

bool aligned(const void *p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

lffw_status from_cuda(cudaError_t err)
{
    if (err == cudaSuccess)
        return LFFW_SUCCESS;
    return err == cudaErrorMemoryAllocation ? LFFW_OUT_OF_MEMORY : LFFW_CUDA_ERROR;
}

lffw_status gate()
{
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) {
        cudaGetLastError();
        return LFFW_CUDA_ERROR;
    }
    return lffw_device_supported(device);
}

bool valid_rows(int64_t rows, int64_t cols, int32_t dtype)
{
    return rows >= 1 && rows <= INT32_MAX && cols >= 8 && cols % 8 == 0 && cols <= lffw::kLayerNormMaxCols &&
           (dtype == LFFW_DT_HALF || dtype == LFFW_DT_BF16);
}

constexpr int64_t kMaxRows = int64_t{1} << 22;
constexpr int64_t kMaxWidth = int64_t{1} << 16;

// Shape, operands and targets, which both directions and the workspace size depend on.
lffw_status validate_vocab(const lffw_vocab_loss_args *a)
{
    if (a == nullptr)
        return LFFW_INVALID_ARGUMENT;
    if (a->struct_size < sizeof(lffw_vocab_loss_args))
        return LFFW_ABI_MISMATCH;
    if (a->rows < 1 || a->rows > kMaxRows || a->vocab < 1 || a->vocab > kMaxRows || a->width < 8 ||
        a->width > kMaxWidth || a->width % 8 != 0 || (a->dtype != LFFW_DT_HALF && a->dtype != LFFW_DT_BF16))
        return LFFW_INVALID_ARGUMENT;
    if (a->x == nullptr || a->weight == nullptr || !aligned(a->x, 16) || !aligned(a->weight, 16))
        return LFFW_INVALID_ARGUMENT;
    if (a->teacher_entries == 0) {
        if (a->labels == nullptr || (a->label_bytes != 4 && a->label_bytes != 8) ||
            !aligned(a->labels, static_cast<uintptr_t>(a->label_bytes)) || a->temperature != 1.0f)
            return LFFW_INVALID_ARGUMENT;
        return LFFW_SUCCESS;
    }
    if (a->teacher_entries < 0 || a->teacher_entries > lffw::kVocabMaxTargets || a->teacher_tokens == nullptr ||
        a->teacher_logits == nullptr || !aligned(a->teacher_tokens, 4))
        return LFFW_INVALID_ARGUMENT;
    if (a->teacher_dtype != LFFW_DT_FLOAT && a->teacher_dtype != LFFW_DT_HALF && a->teacher_dtype != LFFW_DT_BF16)
        return LFFW_INVALID_ARGUMENT;
    if (!aligned(a->teacher_logits, a->teacher_dtype == LFFW_DT_FLOAT ? 4 : 2))
        return LFFW_INVALID_ARGUMENT;
    return std::isfinite(a->temperature) && a->temperature >= 0x1p-6f && a->temperature <= 0x1p6f
               ? LFFW_SUCCESS
               : LFFW_INVALID_ARGUMENT;
}

lffw::VocabLossLaunch vocab_launch(const lffw_vocab_loss_args *a)
{
    lffw::VocabLossLaunch L{};
    L.rows = a->rows;
    L.width = a->width;
    L.vocab = a->vocab;
    L.bf16 = a->dtype == LFFW_DT_BF16;
    L.x = a->x;
    L.weight = a->weight;
    L.labels = a->labels;
    L.label_bytes = a->label_bytes;
    L.ignore_index = a->ignore_index;
    L.targets = a->teacher_entries;
    L.teacher_tokens = a->teacher_tokens;
    L.teacher_logits = a->teacher_logits;
    L.teacher_type = a->teacher_dtype;
    L.temperature = a->temperature;
    L.losses = a->losses;
    L.lse_out = a->lse;
    L.lse_in = a->lse;
    L.dloss = a->dloss;
    L.dx = a->dx;
    L.dweight = a->dweight;
    L.workspace = a->workspace;
    return L;
}

bool workspace_fits(const lffw_vocab_loss_args *a, const lffw::VocabLossLaunch &L, bool grad)
{
    return a->workspace != nullptr && aligned(a->workspace, 256) &&
           a->workspace_bytes >= lffw::vocab_loss_workspace(L, grad);
}

} // namespace

extern "C" {

lffw_status lffw_layer_norm_train(const lffw_layer_norm_train_args *a, void *stream) noexcept
{
    if (a == nullptr)
        return LFFW_INVALID_ARGUMENT;
    if (a->struct_size < sizeof(lffw_layer_norm_train_args))
        return LFFW_ABI_MISMATCH;
    if (!valid_rows(a->rows, a->cols, a->dtype))
        return LFFW_INVALID_ARGUMENT;
    if (a->x == nullptr || a->gamma == nullptr || a->beta == nullptr || a->y == nullptr || a->stats == nullptr ||
        (a->residual != nullptr) != (a->sum_out != nullptr))
        return LFFW_INVALID_ARGUMENT;
    if (!aligned(a->x, 16) || !aligned(a->residual, 16) || !aligned(a->sum_out, 16) || !aligned(a->gamma, 16) ||
        !aligned(a->beta, 16) || !aligned(a->y, 16) || !aligned(a->stats, 4))
        return LFFW_INVALID_ARGUMENT;
    if (!(a->epsilon >= 0.0f) || !std::isfinite(a->epsilon))
        return LFFW_INVALID_ARGUMENT;
    const lffw_status s = gate();
    if (s != LFFW_SUCCESS)
        return s;
    lffw::LayerNormTrainLaunch L{};
    L.rows = a->rows;
    L.cols = a->cols;
    L.bf16 = a->dtype == LFFW_DT_BF16;
    L.x = static_cast<const uint16_t *>(a->x);
    L.residual = static_cast<const uint16_t *>(a->residual);
    L.sum_out = static_cast<uint16_t *>(a->sum_out);
    L.y = static_cast<uint16_t *>(a->y);
    L.gamma = a->gamma;
    L.beta = a->beta;
    L.eps = a->epsilon;
    L.stats = a->stats;
    return from_cuda(lffw::launch_layer_norm_forward(L, static_cast<cudaStream_t>(stream)));
}

int64_t lffw_layer_norm_grad_workspace(int64_t rows, int64_t cols) noexcept
{
    return valid_rows(rows, cols, LFFW_DT_HALF) ? lffw::layer_norm_grad_workspace(rows, cols) : -1;
}

lffw_status lffw_layer_norm_grad(const lffw_layer_norm_grad_args *a, void *stream) noexcept
{
    if (a == nullptr)
        return LFFW_INVALID_ARGUMENT;
    if (a->struct_size < sizeof(lffw_layer_norm_grad_args))
        return LFFW_ABI_MISMATCH;
    if (!valid_rows(a->rows, a->cols, a->dtype))
        return LFFW_INVALID_ARGUMENT;
    if (a->dy == nullptr || a->s == nullptr || a->gamma == nullptr || a->stats == nullptr ||
        (a->dgamma != nullptr) != (a->dbeta != nullptr) || (a->dx == nullptr && a->dgamma == nullptr))
        return LFFW_INVALID_ARGUMENT;
    if (!aligned(a->dy, 16) || !aligned(a->s, 16) || !aligned(a->gamma, 16) || !aligned(a->stats, 4) ||
        !aligned(a->dsum, 16) || !aligned(a->dx, 16) || !aligned(a->dgamma, 4) || !aligned(a->dbeta, 4) ||
        !aligned(a->workspace, 16))
        return LFFW_INVALID_ARGUMENT;
    const lffw_status s = gate();
    if (s != LFFW_SUCCESS)
        return s;
    if (a->dgamma != nullptr) {
        const int64_t need = lffw::layer_norm_grad_workspace(a->rows, a->cols);
        if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < need))
            return LFFW_INVALID_ARGUMENT;
    }
    lffw::LayerNormTrainLaunch L{};
    L.rows = a->rows;
    L.cols = a->cols;
    L.bf16 = a->dtype == LFFW_DT_BF16;
    L.x = static_cast<const uint16_t *>(a->s);
    L.dy = static_cast<const uint16_t *>(a->dy);
    L.gamma = a->gamma;
    L.stats = const_cast<float *>(a->stats);
    L.dsum = static_cast<const uint16_t *>(a->dsum);
    L.dx = static_cast<uint16_t *>(a->dx);
    L.dgamma = a->dgamma;
    L.dbeta = a->dbeta;
    L.workspace = a->workspace;
    return from_cuda(lffw::launch_layer_norm_backward(L, static_cast<cudaStream_t>(stream)));
}

int64_t lffw_vocab_loss_workspace(const lffw_vocab_loss_args *a, int32_t grad) noexcept
{
    return validate_vocab(a) == LFFW_SUCCESS ? lffw::vocab_loss_workspace(vocab_launch(a), grad != 0) : -1;
}

lffw_status lffw_vocab_loss(const lffw_vocab_loss_args *a, void *stream) noexcept
{
    lffw_status s = validate_vocab(a);
    if (s != LFFW_SUCCESS)
        return s;
    if (a->losses == nullptr || a->lse == nullptr || !aligned(a->losses, 4) || !aligned(a->lse, 4))
        return LFFW_INVALID_ARGUMENT;
    if ((s = gate()) != LFFW_SUCCESS)
        return s;
    const lffw::VocabLossLaunch L = vocab_launch(a);
    if (!workspace_fits(a, L, false))
        return LFFW_INVALID_ARGUMENT;
    return from_cuda(lffw::launch_vocab_loss(L, static_cast<cudaStream_t>(stream)));
}

lffw_status lffw_vocab_loss_grad(const lffw_vocab_loss_args *a, void *stream) noexcept
{
    lffw_status s = validate_vocab(a);
    if (s != LFFW_SUCCESS)
        return s;
    if (a->lse == nullptr || a->dloss == nullptr || (a->dx == nullptr && a->dweight == nullptr) ||
        !aligned(a->lse, 4) || !aligned(a->dloss, 4) || !aligned(a->dx, 16) || !aligned(a->dweight, 16))
        return LFFW_INVALID_ARGUMENT;
    if ((s = gate()) != LFFW_SUCCESS)
        return s;
    const lffw::VocabLossLaunch L = vocab_launch(a);
    if (!workspace_fits(a, L, true))
        return LFFW_INVALID_ARGUMENT;
    return from_cuda(lffw::launch_vocab_loss_grad(L, static_cast<cudaStream_t>(stream)));
}

lffw_status lffw_vocab_loss_error(int32_t *code) noexcept
{
    if (code == nullptr)
        return LFFW_INVALID_ARGUMENT;
    const int v = lffw::read_and_clear_token_error();
    if (v < 0) {
        cudaGetLastError();
        return LFFW_CUDA_ERROR;
    }
    *code = v;
    return LFFW_SUCCESS;
}

} // extern "C"
