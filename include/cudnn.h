/*
 * cudnn.h — C ABI of the B200-native convolution-forward and softmax-forward.
 *
 * Drop-in for the MUDA cuDNN shim's hot path: names, argument lists and numeric
 * enum values follow libraries/dnn/include/cudnn.h of the reference (enums
 * cudnn.h:25-128, declarations cudnn.h:150-276).  Enums are int-width.
 * CUDNN_DATA_BFLOAT16 (= 9, NVIDIA's value) is an extension the reference lacks:
 * the reference convolution is fp32-only (cudnn_ops.mm:134-137).
 *
 * Conventions kept from the reference (libraries/dnn/src/cudnn_ops.mm):
 *   - alpha and beta are host float* (cudnn_ops.mm:140-141); beta == 0 means y is not read;
 *   - the convolution workspace is 0 bytes and the algo argument is advisory;
 *   - a KRSC filter is declared with format CUDNN_TENSOR_NHWC, a KCRS filter with NCHW.
 */
#ifndef MUDA_B200_CUDNN_H_
#define MUDA_B200_CUDNN_H_

#include <stddef.h>
#include <stdint.h>
#include <cuda_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

#define CUDNN_MAJOR 8
#define CUDNN_MINOR 9
#define CUDNN_PATCHLEVEL 0
#define CUDNN_VERSION (CUDNN_MAJOR * 1000 + CUDNN_MINOR * 100 + CUDNN_PATCHLEVEL)

typedef enum {
  CUDNN_STATUS_SUCCESS = 0,
  CUDNN_STATUS_NOT_INITIALIZED = 1,
  CUDNN_STATUS_ALLOC_FAILED = 2,
  CUDNN_STATUS_BAD_PARAM = 3,
  CUDNN_STATUS_INTERNAL_ERROR = 4,
  CUDNN_STATUS_INVALID_VALUE = 5,
  CUDNN_STATUS_ARCH_MISMATCH = 6,
  CUDNN_STATUS_MAPPING_ERROR = 7,
  CUDNN_STATUS_EXECUTION_FAILED = 8,
  CUDNN_STATUS_NOT_SUPPORTED = 9
} cudnnStatus_t;

typedef enum {
  CUDNN_DATA_FLOAT = 0,
  CUDNN_DATA_DOUBLE = 1,
  CUDNN_DATA_HALF = 2,
  CUDNN_DATA_INT8 = 3,
  CUDNN_DATA_INT32 = 4,
  CUDNN_DATA_BFLOAT16 = 9 /* extension: not in the reference enum */
} cudnnDataType_t;

typedef enum { CUDNN_TENSOR_NCHW = 0, CUDNN_TENSOR_NHWC = 1 } cudnnTensorFormat_t;

typedef enum { CUDNN_CONVOLUTION = 0, CUDNN_CROSS_CORRELATION = 1 } cudnnConvolutionMode_t;

typedef enum {
  CUDNN_CONVOLUTION_FWD_ALGO_IMPLICIT_GEMM = 0,
  CUDNN_CONVOLUTION_FWD_ALGO_IMPLICIT_PRECOMP_GEMM = 1,
  CUDNN_CONVOLUTION_FWD_ALGO_GEMM = 2,
  CUDNN_CONVOLUTION_FWD_ALGO_DIRECT = 3
} cudnnConvolutionFwdAlgo_t;

typedef enum {
  CUDNN_SOFTMAX_FAST = 0,
  CUDNN_SOFTMAX_ACCURATE = 1,
  CUDNN_SOFTMAX_LOG = 2
} cudnnSoftmaxAlgorithm_t;

typedef enum { CUDNN_SOFTMAX_MODE_INSTANCE = 0, CUDNN_SOFTMAX_MODE_CHANNEL = 1 } cudnnSoftmaxMode_t;

/* reference cudnn.h:72-136 */
typedef enum {
  CUDNN_CONVOLUTION_BWD_DATA_ALGO_0 = 0,
  CUDNN_CONVOLUTION_BWD_DATA_ALGO_1 = 1
} cudnnConvolutionBwdDataAlgo_t;

typedef enum {
  CUDNN_CONVOLUTION_BWD_FILTER_ALGO_0 = 0,
  CUDNN_CONVOLUTION_BWD_FILTER_ALGO_1 = 1
} cudnnConvolutionBwdFilterAlgo_t;

typedef enum {
  CUDNN_ACTIVATION_SIGMOID = 0,
  CUDNN_ACTIVATION_RELU = 1,
  CUDNN_ACTIVATION_TANH = 2,
  CUDNN_ACTIVATION_CLIPPED_RELU = 3,
  CUDNN_ACTIVATION_ELU = 4,
  CUDNN_ACTIVATION_IDENTITY = 5,
  CUDNN_ACTIVATION_SWISH = 6
} cudnnActivationMode_t;

typedef enum { CUDNN_NOT_PROPAGATE_NAN = 0, CUDNN_PROPAGATE_NAN = 1 } cudnnNanPropagation_t;

typedef enum {
  CUDNN_POOLING_MAX = 0,
  CUDNN_POOLING_AVERAGE_COUNT_INCLUDE_PADDING = 1,
  CUDNN_POOLING_AVERAGE_COUNT_EXCLUDE_PADDING = 2,
  CUDNN_POOLING_MAX_DETERMINISTIC = 3
} cudnnPoolingMode_t;

typedef enum {
  CUDNN_BATCHNORM_PER_ACTIVATION = 0,
  CUDNN_BATCHNORM_SPATIAL = 1,
  CUDNN_BATCHNORM_SPATIAL_PERSISTENT = 2
} cudnnBatchNormMode_t;

struct cudnnContext;
struct cudnnTensorStruct;
struct cudnnFilterStruct;
struct cudnnConvolutionStruct;
struct cudnnActivationStruct;
struct cudnnPoolingStruct;
typedef struct cudnnActivationStruct* cudnnActivationDescriptor_t;
typedef struct cudnnPoolingStruct* cudnnPoolingDescriptor_t;
typedef struct cudnnContext* cudnnHandle_t;
typedef struct cudnnTensorStruct* cudnnTensorDescriptor_t;
typedef struct cudnnFilterStruct* cudnnFilterDescriptor_t;
typedef struct cudnnConvolutionStruct* cudnnConvolutionDescriptor_t;

/* Context — reference cudnn_descriptors.mm:46-128 */
size_t cudnnGetVersion(void);
const char* cudnnGetErrorString(cudnnStatus_t status);
cudnnStatus_t cudnnCreate(cudnnHandle_t* handle);
cudnnStatus_t cudnnDestroy(cudnnHandle_t handle);
cudnnStatus_t cudnnSetStream(cudnnHandle_t handle, cudaStream_t streamId);
cudnnStatus_t cudnnGetStream(cudnnHandle_t handle, cudaStream_t* streamId);

/* Tensor descriptors — reference cudnn_descriptors.mm:130-231 */
cudnnStatus_t cudnnCreateTensorDescriptor(cudnnTensorDescriptor_t* tensorDesc);
cudnnStatus_t cudnnSetTensor4dDescriptor(cudnnTensorDescriptor_t tensorDesc,
                                         cudnnTensorFormat_t format, cudnnDataType_t dataType,
                                         int n, int c, int h, int w);
cudnnStatus_t cudnnSetTensor4dDescriptorEx(cudnnTensorDescriptor_t tensorDesc,
                                           cudnnDataType_t dataType, int n, int c, int h, int w,
                                           int nStride, int cStride, int hStride, int wStride);
cudnnStatus_t cudnnGetTensor4dDescriptor(cudnnTensorDescriptor_t tensorDesc,
                                         cudnnDataType_t* dataType, int* n, int* c, int* h, int* w,
                                         int* nStride, int* cStride, int* hStride, int* wStride);
cudnnStatus_t cudnnDestroyTensorDescriptor(cudnnTensorDescriptor_t tensorDesc);

/* Filter descriptors — reference cudnn_descriptors.mm:233-290 */
cudnnStatus_t cudnnCreateFilterDescriptor(cudnnFilterDescriptor_t* filterDesc);
cudnnStatus_t cudnnSetFilter4dDescriptor(cudnnFilterDescriptor_t filterDesc,
                                         cudnnDataType_t dataType, cudnnTensorFormat_t format,
                                         int k, int c, int h, int w);
cudnnStatus_t cudnnGetFilter4dDescriptor(cudnnFilterDescriptor_t filterDesc,
                                         cudnnDataType_t* dataType, cudnnTensorFormat_t* format,
                                         int* k, int* c, int* h, int* w);
cudnnStatus_t cudnnDestroyFilterDescriptor(cudnnFilterDescriptor_t filterDesc);

/* Convolution descriptors — reference cudnn_descriptors.mm:292-385 */
cudnnStatus_t cudnnCreateConvolutionDescriptor(cudnnConvolutionDescriptor_t* convDesc);
cudnnStatus_t cudnnSetConvolution2dDescriptor(cudnnConvolutionDescriptor_t convDesc, int pad_h,
                                              int pad_w, int u, int v, int dilation_h,
                                              int dilation_w, cudnnConvolutionMode_t mode,
                                              cudnnDataType_t computeType);
cudnnStatus_t cudnnSetConvolutionGroupCount(cudnnConvolutionDescriptor_t convDesc, int groupCount);
cudnnStatus_t cudnnGetConvolutionGroupCount(cudnnConvolutionDescriptor_t convDesc, int* groupCount);
cudnnStatus_t cudnnGetConvolution2dForwardOutputDim(cudnnConvolutionDescriptor_t convDesc,
                                                    cudnnTensorDescriptor_t inputTensorDesc,
                                                    cudnnFilterDescriptor_t filterDesc, int* n,
                                                    int* c, int* h, int* w);
cudnnStatus_t cudnnDestroyConvolutionDescriptor(cudnnConvolutionDescriptor_t convDesc);

/* Activation and pooling descriptors — reference cudnn_descriptors.mm:382-484 */
cudnnStatus_t cudnnCreateActivationDescriptor(cudnnActivationDescriptor_t* activationDesc);
cudnnStatus_t cudnnSetActivationDescriptor(cudnnActivationDescriptor_t activationDesc,
                                           cudnnActivationMode_t mode,
                                           cudnnNanPropagation_t reluNanOpt, double coef);
cudnnStatus_t cudnnGetActivationDescriptor(cudnnActivationDescriptor_t activationDesc,
                                           cudnnActivationMode_t* mode,
                                           cudnnNanPropagation_t* reluNanOpt, double* coef);
cudnnStatus_t cudnnDestroyActivationDescriptor(cudnnActivationDescriptor_t activationDesc);
cudnnStatus_t cudnnCreatePoolingDescriptor(cudnnPoolingDescriptor_t* poolingDesc);
cudnnStatus_t cudnnSetPooling2dDescriptor(cudnnPoolingDescriptor_t poolingDesc,
                                          cudnnPoolingMode_t mode,
                                          cudnnNanPropagation_t maxpoolingNanOpt, int windowHeight,
                                          int windowWidth, int verticalPadding,
                                          int horizontalPadding, int verticalStride,
                                          int horizontalStride);
cudnnStatus_t cudnnGetPooling2dForwardOutputDim(cudnnPoolingDescriptor_t poolingDesc,
                                                cudnnTensorDescriptor_t inputTensorDesc, int* n,
                                                int* c, int* h, int* w);
cudnnStatus_t cudnnDestroyPoolingDescriptor(cudnnPoolingDescriptor_t poolingDesc);
/* reference cudnn_descriptors.mm:486-500 */
cudnnStatus_t cudnnDeriveBNTensorDescriptor(cudnnTensorDescriptor_t derivedBnDesc,
                                            cudnnTensorDescriptor_t xDesc,
                                            cudnnBatchNormMode_t mode);

/* Operations — reference cudnn_ops.mm:89-193 (conv) and cudnn_ops.mm:625-720 (softmax) */
cudnnStatus_t cudnnGetConvolutionForwardWorkspaceSize(
    cudnnHandle_t handle, cudnnTensorDescriptor_t xDesc, cudnnFilterDescriptor_t wDesc,
    cudnnConvolutionDescriptor_t convDesc, cudnnTensorDescriptor_t yDesc,
    cudnnConvolutionFwdAlgo_t algo, size_t* sizeInBytes);
cudnnStatus_t cudnnConvolutionForward(cudnnHandle_t handle, const void* alpha,
                                      cudnnTensorDescriptor_t xDesc, const void* x,
                                      cudnnFilterDescriptor_t wDesc, const void* w,
                                      cudnnConvolutionDescriptor_t convDesc,
                                      cudnnConvolutionFwdAlgo_t algo, void* workSpace,
                                      size_t workSpaceSizeInBytes, const void* beta,
                                      cudnnTensorDescriptor_t yDesc, void* y);
cudnnStatus_t cudnnSoftmaxForward(cudnnHandle_t handle, cudnnSoftmaxAlgorithm_t algo,
                                  cudnnSoftmaxMode_t mode, const void* alpha,
                                  cudnnTensorDescriptor_t xDesc, const void* x, const void* beta,
                                  cudnnTensorDescriptor_t yDesc, void* y);

/* Neighbours of the convolution, fp32 — reference cudnn_ops.mm:195-624, 722-902.
 * Backward data, AddTensor, ReLU / clipped ReLU / identity and pooling give the
 * reference's per-output arithmetic exactly; the reductions (backward filter and
 * bias, batch-norm training statistics) are deterministic but summed in a
 * different order than the reference's single sequential loop.  The algo and
 * workspace arguments of the backward calls are ignored: the backward filter's
 * partial sums live in the handle's workspace. */
cudnnStatus_t cudnnConvolutionBackwardData(cudnnHandle_t handle, const void* alpha,
                                           cudnnFilterDescriptor_t wDesc, const void* w,
                                           cudnnTensorDescriptor_t dyDesc, const void* dy,
                                           cudnnConvolutionDescriptor_t convDesc,
                                           cudnnConvolutionBwdDataAlgo_t algo, void* workSpace,
                                           size_t workSpaceSizeInBytes, const void* beta,
                                           cudnnTensorDescriptor_t dxDesc, void* dx);
cudnnStatus_t cudnnConvolutionBackwardFilter(cudnnHandle_t handle, const void* alpha,
                                             cudnnTensorDescriptor_t xDesc, const void* x,
                                             cudnnTensorDescriptor_t dyDesc, const void* dy,
                                             cudnnConvolutionDescriptor_t convDesc,
                                             cudnnConvolutionBwdFilterAlgo_t algo, void* workSpace,
                                             size_t workSpaceSizeInBytes, const void* beta,
                                             cudnnFilterDescriptor_t dwDesc, void* dw);
cudnnStatus_t cudnnConvolutionBackwardBias(cudnnHandle_t handle, const void* alpha,
                                           cudnnTensorDescriptor_t dyDesc, const void* dy,
                                           const void* beta, cudnnTensorDescriptor_t dbDesc,
                                           void* db);
cudnnStatus_t cudnnAddTensor(cudnnHandle_t handle, const void* alpha, cudnnTensorDescriptor_t aDesc,
                             const void* A, const void* beta, cudnnTensorDescriptor_t cDesc,
                             void* C);
cudnnStatus_t cudnnActivationForward(cudnnHandle_t handle,
                                     cudnnActivationDescriptor_t activationDesc, const void* alpha,
                                     cudnnTensorDescriptor_t xDesc, const void* x, const void* beta,
                                     cudnnTensorDescriptor_t yDesc, void* y);
cudnnStatus_t cudnnPoolingForward(cudnnHandle_t handle, cudnnPoolingDescriptor_t poolingDesc,
                                  const void* alpha, cudnnTensorDescriptor_t xDesc, const void* x,
                                  const void* beta, cudnnTensorDescriptor_t yDesc, void* y);
cudnnStatus_t cudnnBatchNormalizationForwardInference(
    cudnnHandle_t handle, cudnnBatchNormMode_t mode, const void* alpha, const void* beta,
    cudnnTensorDescriptor_t xDesc, const void* x, cudnnTensorDescriptor_t yDesc, void* y,
    cudnnTensorDescriptor_t bnScaleBiasMeanVarDesc, const void* bnScale, const void* bnBias,
    const void* estimatedMean, const void* estimatedVariance, double epsilon);
cudnnStatus_t cudnnBatchNormalizationForwardTraining(
    cudnnHandle_t handle, cudnnBatchNormMode_t mode, const void* alpha, const void* beta,
    cudnnTensorDescriptor_t xDesc, const void* x, cudnnTensorDescriptor_t yDesc, void* y,
    cudnnTensorDescriptor_t bnScaleBiasMeanVarDesc, const void* bnScale, const void* bnBias,
    double exponentialAverageFactor, void* resultRunningMean, void* resultRunningVariance,
    double epsilon, void* resultSaveMean, void* resultSaveInvVariance);

/* Losses over a linear head's vocabulary, forward and with gradients (extensions).
 *
 * x holds T tokens of H features: a tensor descriptor with c = H, cStride 1 and its
 * (n, h, w) positions a uniform stride apart.  w is the head: a 1x1 filter, k = V words
 * of c = H features.  Both BFLOAT16 or both HALF; z = x w^T / temperature and everything
 * computed from it is fp32 until a 16-bit output.  The T x V logits are never stored.
 *
 *   cross entropy   loss[t] = lse(z[t]) - z[t][labels[t]]
 *   distillation    q = softmax(teacherLogits[t] / temperature) over the row's topK
 *                   (1..256) entries, loss[t] = sum_k q_k (log q_k - (z[t][index_k] - lse))
 *
 * A negative label leaves its token out; a negative teacher index, or a teacher logit of
 * -inf, leaves its entry out, and a token without entries is left out.  A token that is
 * left out has loss 0, logSumExp 0 and no gradient, whatever its x and dloss hold.
 * Temperatures are 2^-64 to 2^64.  Equal indices of a token add up.  A label or index of V or
 * more makes its token's loss, and the gradients it enters, NaN.  labels and teacherIndex [T][topK] are int64 (as
 * training programs hold them); teacherLogits [T][topK], loss and logSumExp are float.
 *
 * Backward computes the gradients of sum_t dloss[t] * loss[t] in one pass over the
 * tokens; it computes the losses too and writes them when loss / logSumExp are not null,
 * so a training step whose dloss is known needs no Forward.  dx (like x; it may be x
 * itself) or dw (like w) may be null with its descriptor: it is not computed.  Results
 * do not depend on the stream's other work: no atomics.  The gradient of the logits is
 * rounded to 16 bits on its way into both products; what that leaves is added to both for up
 * to 64 tokens, and to dx at the target words of tokens with up to four of them.  In HALF it
 * is scaled by one power of two per piece of the tokens (below), so tokens whose |dloss| is
 * 2^-20 of their piece's largest or less keep fewer bits of it.
 *
 * The workspace: null uses the handle's own (grown to what GetWorkspaceSize reports).  A
 * call runs over pieces of the tokens that need at most 2 GiB for 16-bit numerators and
 * 1 GiB for what else grows with their number (128 tokens at least, which need more only
 * beyond 8 million words); gradients of several pieces need V*H floats too, and a w whose rows
 * are not a multiple of 16 bytes a copy of it.  The size reported serves either or both
 * gradients and x and w at any address.  A workspace given (aligned to 256 bytes) bounds the
 * memory instead: smaller ones mean smaller pieces, down to 128 tokens, and a copy of w in
 * slices of 16 MiB; BAD_PARAM below that.
 * Calls on a handle wait for its workspace across streams.  Under stream capture null takes an
 * allocation of the graph's own instead (a memory node, with CUDA's limits on such graphs), so
 * replays share nothing with the handle; a workspace given is the caller's to keep and order.
 */
cudnnStatus_t cudnnGetLinearCrossEntropyWorkspaceSize(cudnnHandle_t handle,
                                                      cudnnTensorDescriptor_t xDesc,
                                                      cudnnFilterDescriptor_t wDesc, int gradients,
                                                      size_t* sizeInBytes);
cudnnStatus_t cudnnLinearCrossEntropyForward(cudnnHandle_t handle, cudnnTensorDescriptor_t xDesc,
                                             const void* x, cudnnFilterDescriptor_t wDesc,
                                             const void* w, const int64_t* labels, void* workSpace,
                                             size_t workSpaceSizeInBytes, float* loss,
                                             float* logSumExp);
cudnnStatus_t cudnnLinearCrossEntropyBackward(cudnnHandle_t handle, cudnnTensorDescriptor_t xDesc,
                                              const void* x, cudnnFilterDescriptor_t wDesc,
                                              const void* w, const int64_t* labels,
                                              const float* dloss, void* workSpace,
                                              size_t workSpaceSizeInBytes, float* loss,
                                              float* logSumExp, cudnnTensorDescriptor_t dxDesc,
                                              void* dx, cudnnFilterDescriptor_t dwDesc, void* dw);
cudnnStatus_t cudnnGetLinearDistillationWorkspaceSize(cudnnHandle_t handle,
                                                      cudnnTensorDescriptor_t xDesc,
                                                      cudnnFilterDescriptor_t wDesc, int topK,
                                                      int gradients, size_t* sizeInBytes);
cudnnStatus_t cudnnLinearDistillationForward(cudnnHandle_t handle, cudnnTensorDescriptor_t xDesc,
                                             const void* x, cudnnFilterDescriptor_t wDesc,
                                             const void* w, int topK, const int64_t* teacherIndex,
                                             const float* teacherLogits, double temperature,
                                             void* workSpace, size_t workSpaceSizeInBytes,
                                             float* loss, float* logSumExp);
cudnnStatus_t cudnnLinearDistillationBackward(cudnnHandle_t handle, cudnnTensorDescriptor_t xDesc,
                                              const void* x, cudnnFilterDescriptor_t wDesc,
                                              const void* w, int topK, const int64_t* teacherIndex,
                                              const float* teacherLogits, double temperature,
                                              const float* dloss, void* workSpace,
                                              size_t workSpaceSizeInBytes, float* loss,
                                              float* logSumExp, cudnnTensorDescriptor_t dxDesc,
                                              void* dx, cudnnFilterDescriptor_t dwDesc, void* dw);

/* Losses of post-training on the same head (extensions).  nll[t] is the cross entropy above,
 * the negative log-probability of the label; x, w, labels, the workspace, streams and capture
 * are as above, and so is a token that a negative label leaves out: 0 in every output, no
 * gradient, whatever the other inputs hold there.  nll is 0 or more, at any temperature.  All
 * float arrays are fp32.  Device memory is the current device's: another one's is BAD_PARAM.
 *
 * Policy loss, per token, z = x w^T / temperature:
 *   ratio = exp(oldNll - nll)            oldNll null: 1, and its gradient as if it were nll
 *   gain  = min(ratio A, clip(ratio, 1 - clipLow, 1 + clipHigh) A)    A = advantages[t]
 *           where A < 0 and dualClip >= 1 (0: off): max(gain, dualClip A)
 *   kl    = exp(d) - d - 1, d = nll - refNll                refNll null: 0, klCoef 0
 *   loss  = klCoef kl - gain
 * The gradient is that of the side that min (or max) took, of ratio A where they are equal.
 * A token whose advantage is 0 has gain 0 at any ratio.  clipLow is 0 to 1, clipHigh, dualClip
 * and klCoef at most 2^64.
 *
 * Preference loss of pairs of sequences: sequence s holds the rows offsets[s] to
 * offsets[s + 1] - 1 (int64 on the device, 2 * pairs + 1 of them, ascending from 0 at least to T at
 * most); sequence p is the chosen one of pair p, pairs + p the rejected one.
 *   L[s] = sum of refNll - nll over the tokens of s that are not left out (refNll null: 0),
 *          with `averaged` divided by their number
 *   h    = beta (L[p] - L[pairs + p]) - margin
 *   loss[p] = SIGMOID: softplus(-h) + labelSmoothing h; HINGE: max(0, 1 - h);
 *             SQUARED: ((h - 1/2) / beta)^2
 *   rewards[s] = beta L[s]
 * An infinite h (a reference that did not know a token) has the loss that is its limit.
 * beta is 2^-64 to 2^64, labelSmoothing 0 to 1/2 and 0 for the other modes.  A pair with a
 * sequence of which no token is kept is left out: loss and rewards 0, no gradient.  Rows of no
 * sequence have an nll and no gradient.  A pair whose offsets do not ascend within 0..T has NaN
 * for its loss and rewards and no gradient of its own.
 *
 * A label of V or more makes its token's outputs NaN, its pair's, and the gradients they enter.
 * Every output may be null (Forward: not all of them).  Backward computes the outputs too, and
 * the gradients of sum dloss * loss: dloss holds T floats for a policy loss, `pairs` for a
 * preference loss.  Logits are computed once, but for preference gradients of more tokens than
 * one piece has: a pair's loss takes all its tokens, so each piece's logits are computed again
 * after them.  To that end a piece of a preference's holds up to 4 GiB of numerators (not 2, see
 * the workspace above); 8 bytes per token come besides.  A preference's gradients of more than 64
 * tokens are scaled on their way into dw in BFLOAT16 as well, and in both types by the power of
 * two above or less, down to half of it: a sequence's tokens share one gradient, and the factor
 * that leaves least of it to rounding is taken. */
typedef enum {
  CUDNN_PREFERENCE_SIGMOID = 0,
  CUDNN_PREFERENCE_HINGE = 1,
  CUDNN_PREFERENCE_SQUARED = 2,
} cudnnPreferenceMode_t;

cudnnStatus_t cudnnGetLinearPolicyLossWorkspaceSize(cudnnHandle_t handle,
                                                    cudnnTensorDescriptor_t xDesc,
                                                    cudnnFilterDescriptor_t wDesc, int gradients,
                                                    size_t* sizeInBytes);
cudnnStatus_t cudnnLinearPolicyLossForward(
    cudnnHandle_t handle, cudnnTensorDescriptor_t xDesc, const void* x,
    cudnnFilterDescriptor_t wDesc, const void* w, const int64_t* labels, const float* oldNll,
    const float* refNll, const float* advantages, double temperature, double clipLow,
    double clipHigh, double dualClip, double klCoef, void* workSpace, size_t workSpaceSizeInBytes,
    float* loss, float* nll, float* ratio, float* kl);
cudnnStatus_t cudnnLinearPolicyLossBackward(
    cudnnHandle_t handle, cudnnTensorDescriptor_t xDesc, const void* x,
    cudnnFilterDescriptor_t wDesc, const void* w, const int64_t* labels, const float* oldNll,
    const float* refNll, const float* advantages, double temperature, double clipLow,
    double clipHigh, double dualClip, double klCoef, const float* dloss, void* workSpace,
    size_t workSpaceSizeInBytes, float* loss, float* nll, float* ratio, float* kl,
    cudnnTensorDescriptor_t dxDesc, void* dx, cudnnFilterDescriptor_t dwDesc, void* dw);
cudnnStatus_t cudnnGetLinearPreferenceLossWorkspaceSize(cudnnHandle_t handle,
                                                        cudnnTensorDescriptor_t xDesc,
                                                        cudnnFilterDescriptor_t wDesc,
                                                        int gradients, size_t* sizeInBytes);
cudnnStatus_t cudnnLinearPreferenceLossForward(
    cudnnHandle_t handle, cudnnTensorDescriptor_t xDesc, const void* x,
    cudnnFilterDescriptor_t wDesc, const void* w, const int64_t* labels, int pairs,
    const int64_t* offsets, const float* refNll, cudnnPreferenceMode_t mode, int averaged,
    double beta, double margin, double labelSmoothing, void* workSpace,
    size_t workSpaceSizeInBytes, float* loss, float* rewards, float* nll);
cudnnStatus_t cudnnLinearPreferenceLossBackward(
    cudnnHandle_t handle, cudnnTensorDescriptor_t xDesc, const void* x,
    cudnnFilterDescriptor_t wDesc, const void* w, const int64_t* labels, int pairs,
    const int64_t* offsets, const float* refNll, cudnnPreferenceMode_t mode, int averaged,
    double beta, double margin, double labelSmoothing, const float* dloss, void* workSpace,
    size_t workSpaceSizeInBytes, float* loss, float* rewards, float* nll,
    cudnnTensorDescriptor_t dxDesc, void* dx, cudnnFilterDescriptor_t dwDesc, void* dw);

/* Embeddings (extensions): a table w of V words, a 1x1 filter (k = V, c = H features) as for
 * the head above, and tokens (int64, one per row of y or dy; rows as x above).
 *
 *   Forward    y[t] = alpha w[tokens[t]] + beta y[t]
 *   Backward   dw[v] = alpha sum of dy[t] over the rows with tokens[t] == v, + beta dw[v]
 *
 * Table and rows are of one type (FLOAT, HALF or BFLOAT16), or a FLOAT table has 16-bit rows.
 * alpha and beta are floats on the host; beta 0 does not read y or dw; sums are fp32 and round
 * once.  Backward with beta 1 touches only the rows of words that occur (the second micro-batch
 * of a step, or a table that is also the head, whose dw the losses above have written), others
 * write all V rows.
 *
 * A negative token (padding) stands for a row of zeros: y[t] = beta y[t], and its dy is not
 * read.  A token of V or more makes its row of y NaN and enters no gradient.  A word's rows are
 * added in the order of their positions: results are the same on every run.
 *
 * Device memory is the current device's: another one's is BAD_PARAM.  Backward's workspace: null
 * uses the handle's own, ordered and captured as for the losses above; GetWorkspaceSize reports
 * what a given one (aligned to 256 bytes) needs. */
cudnnStatus_t cudnnEmbeddingForward(cudnnHandle_t handle, const void* alpha,
                                    cudnnFilterDescriptor_t wDesc, const void* w,
                                    const int64_t* tokens, const void* beta,
                                    cudnnTensorDescriptor_t yDesc, void* y);
cudnnStatus_t cudnnGetEmbeddingBackwardWorkspaceSize(cudnnHandle_t handle,
                                                     cudnnTensorDescriptor_t dyDesc,
                                                     cudnnFilterDescriptor_t dwDesc,
                                                     size_t* sizeInBytes);
cudnnStatus_t cudnnEmbeddingBackward(cudnnHandle_t handle, const void* alpha,
                                     cudnnTensorDescriptor_t dyDesc, const void* dy,
                                     const int64_t* tokens, void* workSpace,
                                     size_t workSpaceSizeInBytes, const void* beta,
                                     cudnnFilterDescriptor_t dwDesc, void* dw);

#ifdef __cplusplus
}
#endif

#endif /* MUDA_B200_CUDNN_H_ */
