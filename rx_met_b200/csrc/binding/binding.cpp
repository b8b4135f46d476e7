// Torch side of the hot entry points: argument checks, output allocation, workspace and stream lookup, the call into
// the C ABI of librxmet_b200.so and the autograd node of the learned-grid quantize-dequantize.
//
// In Python with ctypes these took 60 to 180 us a call (qdq 4096 x 4096 with its gradients 160 us against 67 us of
// kernels, one GRU inference 92 us against 72), so that the small calls were bound by the interpreter.  The C ABI is
// not linked: the package loads the library globally first, so that an overridden library path reaches this module too.
#include <ATen/core/Tensor.h>
#include <ATen/ops/clamp.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <array>
#include <cstring>
#include <map>
#include <mutex>
#include <optional>
#include <vector>

#include "rxmet_b200.h"
#include "rxmet_b200_lstm.h"
#include "rxmet_b200_mixer.h"

namespace {

using at::Tensor;
using MaybeTensor = std::optional<Tensor>;
using Shape = std::vector<int64_t>;

void *streamOf(const Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// Null for an absent or empty tensor, as the C ABI expects.
template <class T>
T *pointer(const Tensor &t) {
    return t.defined() && t.numel() > 0 ? static_cast<T *>(t.data_ptr()) : nullptr;
}

std::string listText(at::IntArrayRef sizes) {
    std::string text = "[";
    for (size_t i = 0; i < sizes.size(); ++i) text += (i ? ", " : "") + std::to_string(sizes[i]);
    return text + "]";
}

Tensor emptyLike(const Tensor &like, at::IntArrayRef shape, at::ScalarType type = at::kFloat) {
    return at::empty(shape, at::TensorOptions().dtype(type).device(like.device()));
}

// Tensors of the given shapes over ONE allocation, each on a 16-byte boundary: a forward returns sixteen small tensors,
// and an allocator round trip for each is host time on the critical path of a training step.
std::vector<Tensor> carve(const Tensor &like, at::ScalarType type, const std::vector<Shape> &shapes) {
    const int64_t per = 16 / static_cast<int64_t>(c10::elementSize(type));
    std::vector<int64_t> offsets;
    int64_t total = 0;
    for (const Shape &shape : shapes) {
        int64_t n = 1;
        for (int64_t d : shape) n *= d;
        offsets.push_back(total);
        total += (n + per - 1) / per * per;
    }
    const Tensor pool = emptyLike(like, {std::max<int64_t>(total, 1)}, type);
    std::vector<Tensor> out;
    out.reserve(shapes.size());
    for (size_t i = 0; i < shapes.size(); ++i) {
        Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(pool.storage()), pool.key_set(), pool.dtype());
        t.unsafeGetTensorImpl()->set_storage_offset(pool.storage_offset() + offsets[i]);
        t.unsafeGetTensorImpl()->set_sizes_contiguous(shapes[i]);
        out.push_back(std::move(t));
    }
    return out;
}

// One growing scratch buffer per device and stream, reused across calls (calls on one stream follow one another).
Tensor workspace(const c10::Device &device, int64_t bytes) {
    static std::mutex mutex;
    static auto &buffers = *new std::map<std::pair<int, void *>, Tensor>;   // outlives the CUDA context's teardown
    void *stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    std::lock_guard<std::mutex> lock(mutex);
    Tensor &have = buffers[{device.index(), stream}];
    if (!have.defined() || have.numel() < bytes) {
        have = Tensor();
        have = at::empty({std::max<int64_t>(bytes, 1 << 20)}, at::TensorOptions().dtype(at::kByte).device(device));
    }
    return have;
}

// ---- GRU ----------------------------------------------------------------------------------------------------------

Tensor floatCuda(const Tensor &t, const char *name, at::IntArrayRef shape) {
    if (!t.is_cuda() || t.scalar_type() != at::kFloat) TORCH_CHECK(false, name, " must be CUDA float32 tensor");
    if (t.sizes() != shape) TORCH_CHECK(false, name, " must have shape ", listText(shape));
    return t.contiguous();
}

// Status of the library and the 18 tensors of the interface: h, v, five code tensors, eleven masks.
std::pair<int, std::vector<Tensor>> gruForwardQuant(bool training, int T, int B, int I, int H, Tensor W, Tensor R, Tensor bw,
                                                    Tensor br, Tensor x, const MaybeTensor &h0, uintptr_t paramsAddress,
                                                    bool floatCarrier) {
    const int64_t C = 3 * static_cast<int64_t>(H);
    W = floatCuda(W, "W", {I, C});
    R = floatCuda(R, "R", {H, C});
    bw = floatCuda(bw, "bw", {C});
    br = floatCuda(br, "br", {C});
    x = floatCuda(x, "x", {T, B, I});
    Tensor h0v;
    if (h0 && h0->numel() > 0) h0v = floatCuda(*h0, "h0", {B, H});
    const c10::cuda::CUDAGuard guard(x.device());
    std::vector<Tensor> out{emptyLike(x, {T + 1, B, H}), emptyLike(x, {T, B, 4 * static_cast<int64_t>(H)})};
    for (Tensor &t : carve(x, at::kInt, {{I, C}, {H, C}, {C}, {C}, {T, B, I}})) out.push_back(std::move(t));
    rxmet_gru_masks masks{};
    if (training) {
        uint8_t **const fields[] = {&masks.x, &masks.h0, &masks.W, &masks.R, &masks.bw, &masks.br, &masks.weight_ih_linear,
                                    &masks.weight_hh_linear, &masks.gate_input, &masks.gate_output, &masks.h};
        std::vector<Shape> shapes{{T, B, I}, {B, H}, {I, C}, {H, C}, {C}, {C}, {T, B, C}, {T, B, C}, {T, B, C}, {T, B, C}, {T, B, H}};
        if (!h0v.defined()) shapes[1] = {0};
        size_t k = 0;
        for (Tensor &t : carve(x, at::kByte, shapes)) {
            *fields[k++] = pointer<uint8_t>(t);
            out.push_back(std::move(t));
        }
    } else {
        const Tensor none = emptyLike(x, {0}, at::kByte);
        out.resize(18, none);
    }
    const Tensor ws = workspace(x.device(), static_cast<int64_t>(rxmet_gru_workspace_bytes(1, T, B, I, H)));
    const auto *params = reinterpret_cast<const rxmet_gru_quant_params *>(paramsAddress);
    const auto entry = floatCarrier ? rxmet_gru_forward_quant_fp_carrier : rxmet_gru_forward_quant;
    const pybind11::gil_scoped_release release;
    const int status = entry(training, T, B, I, H, pointer<float>(W), pointer<float>(R), pointer<float>(bw), pointer<float>(br),
                             pointer<float>(x), pointer<float>(h0v), params, pointer<float>(out[0]), pointer<float>(out[1]),
                             pointer<int32_t>(out[2]), pointer<int32_t>(out[3]), pointer<int32_t>(out[4]),
                             pointer<int32_t>(out[5]), pointer<int32_t>(out[6]), nullptr, nullptr, training ? &masks : nullptr,
                             ws.data_ptr(), static_cast<size_t>(ws.numel()), streamOf(x));
    return {status, std::move(out)};
}

std::pair<int, std::vector<Tensor>> gruBackwardQuant(int T, int B, int I, int H, const std::array<Tensor, 5> &cached, Tensor dh,
                                                     Tensor h, Tensor v, uintptr_t paramsAddress,
                                                     const std::array<MaybeTensor, 11> &flags) {
    const int64_t C = 3 * static_cast<int64_t>(H);
    const char *const names[] = {"W_q", "R_q", "bw_q", "br_q", "x_q"};
    const Shape shapes[] = {{I, C}, {H, C}, {C}, {C}, {T, B, I}};
    std::array<Tensor, 5> codes;
    for (int k = 0; k < 5; ++k) {
        if (!cached[k].is_cuda() || cached[k].sizes() != at::IntArrayRef(shapes[k]))
            TORCH_CHECK(false, names[k], " must be a CUDA tensor of shape ", listText(shapes[k]));
        codes[k] = (cached[k].scalar_type() == at::kInt ? cached[k] : cached[k].to(at::kInt)).contiguous();
    }
    dh = floatCuda(dh, "dh_new", {T + 1, B, H});
    h = floatCuda(h, "h", {T + 1, B, H});
    v = floatCuda(v, "v", {T, B, 4 * static_cast<int64_t>(H)});
    rxmet_gru_masks masks{};
    uint8_t **const fields[] = {&masks.x, &masks.h0, &masks.W, &masks.R, &masks.bw, &masks.br, &masks.weight_ih_linear,
                                &masks.weight_hh_linear, &masks.gate_input, &masks.gate_output, &masks.h};
    std::array<Tensor, 11> live;
    for (int k = 0; k < 11; ++k) {
        if (!flags[k] || flags[k]->numel() == 0) continue;
        live[k] = flags[k]->contiguous();
        *fields[k] = static_cast<uint8_t *>(live[k].data_ptr());
    }
    const c10::cuda::CUDAGuard guard(h.device());
    std::vector<Tensor> out = carve(h, at::kFloat, {{T, B, I}, {I, C}, {H, C}, {C}, {C}, {B, H}});
    const auto *params = reinterpret_cast<const rxmet_gru_quant_params *>(paramsAddress);
    const int8_t *bits = params->config.bits;
    const bool tensorCores = bits[RXMET_GRU_W] <= 8 && bits[RXMET_GRU_R] <= 8 && bits[RXMET_GRU_X] <= 16 && bits[RXMET_GRU_H] <= 16;
    const Tensor ws = workspace(h.device(), static_cast<int64_t>(rxmet_gru_workspace_bytes(tensorCores ? 2 : 4, T, B, I, H)));
    const pybind11::gil_scoped_release release;
    const int status = rxmet_gru_backward_quant(
        T, B, I, H, pointer<int32_t>(codes[0]), pointer<int32_t>(codes[1]), pointer<int32_t>(codes[2]), pointer<int32_t>(codes[3]),
        pointer<int32_t>(codes[4]), pointer<float>(dh), pointer<float>(h), pointer<float>(v), params, &masks,
        pointer<float>(out[0]), pointer<float>(out[1]), pointer<float>(out[2]), pointer<float>(out[3]), pointer<float>(out[4]),
        pointer<float>(out[5]), ws.data_ptr(), static_cast<size_t>(ws.numel()), streamOf(h));
    return {status, std::move(out)};
}

// ---- LSTM ---------------------------------------------------------------------------------------------------------

constexpr int kMasters = 7, kTrace = 7;

Tensor lstmFloat(const Tensor &t, const char *name) {
    if (t.scalar_type() != at::kFloat) TORCH_CHECK(false, name, " must be a float32 tensor");
    if (!t.is_cuda()) TORCH_CHECK(false, name, " must be a CUDA tensor");
    return t.contiguous();
}

// Checked, contiguous arguments of a forward or backward call (absent ones stay undefined).
struct LstmInputs {
    Tensor x, wIh, wHh, bIh, bHh, h0, c0;
    int T, B, I, H;
    LstmInputs(const Tensor &input, const Tensor &weightIh, const Tensor &weightHh, const MaybeTensor &biasIh,
               const MaybeTensor &biasHh, const MaybeTensor &hidden, const MaybeTensor &cell, bool batchFirst) {
        x = lstmFloat(input, "input");
        TORCH_CHECK(x.dim() == 3, "input must have 3 dimensions");
        if (batchFirst) x = x.transpose(0, 1).contiguous();
        T = static_cast<int>(x.size(0)); B = static_cast<int>(x.size(1)); I = static_cast<int>(x.size(2));
        wIh = lstmFloat(weightIh, "weight_ih");
        wHh = lstmFloat(weightHh, "weight_hh");
        TORCH_CHECK(wIh.dim() == 2 && wHh.dim() == 2 && wIh.size(0) % 4 == 0, "weights must be [4H, I] and [4H, H]");
        H = static_cast<int>(wIh.size(0) / 4);
        TORCH_CHECK(wIh.size(1) == I && wHh.size(0) == 4 * static_cast<int64_t>(H) && wHh.size(1) == H,
                    "weight shapes do not match input_size / hidden_size");
        TORCH_CHECK(biasIh.has_value() == biasHh.has_value(), "bias_ih and bias_hh must be given together");
        if (biasIh) {
            bIh = lstmFloat(*biasIh, "bias_ih");
            bHh = lstmFloat(*biasHh, "bias_hh");
            for (const Tensor *b : {&bIh, &bHh}) TORCH_CHECK(b->dim() == 1 && b->size(0) == 4 * static_cast<int64_t>(H), "bias must be [4H]");
        }
        TORCH_CHECK(hidden.has_value() == cell.has_value(), "initial_hidden and initial_cell must be given together");
        if (hidden) {
            h0 = lstmFloat(*hidden, "initial_hidden").reshape({B, H});
            c0 = lstmFloat(*cell, "initial_cell").reshape({B, H});
        }
    }
};

using LstmForward = std::tuple<int, Tensor, Tensor, Tensor, std::vector<Tensor>, std::vector<Tensor>, std::vector<Tensor>, std::vector<Tensor>>;

LstmForward lstmForwardQuant(const Tensor &input, const Tensor &weightIh, const Tensor &weightHh, const MaybeTensor &biasIh,
                             const MaybeTensor &biasHh, const MaybeTensor &hidden, const MaybeTensor &cell, bool batchFirst,
                             uintptr_t paramsAddress, bool requireExact, bool checkpoints) {
    const LstmInputs p(input, weightIh, weightHh, biasIh, biasHh, hidden, cell, batchFirst);
    const auto *params = reinterpret_cast<const rxmet_lstm_quant_params *>(paramsAddress);
    const int64_t T = p.T, B = p.B, H = p.H;
    TORCH_CHECK(params->input_size == p.I && params->hidden_size == p.H,
                "quantization parameters do not match input_size / hidden_size of the module");
    TORCH_CHECK((params->bias_enabled != 0) == p.bIh.defined(), "quantization parameters do not match the bias setting of the module");
    const c10::cuda::CUDAGuard guard(p.x.device());
    const Tensor out = emptyLike(p.x, {T, B, H}), hn = emptyLike(p.x, {1, B, H}), cn = emptyLike(p.x, {1, B, H});
    std::vector<Tensor> values, clamped, masters, masterClamped;
    rxmet_lstm_trace trace{};
    rxmet_lstm_masters saved{};
    static_assert(sizeof(trace) == 2 * kTrace * sizeof(void *) && sizeof(saved) == 2 * kMasters * sizeof(void *), "pointer tables");
    if (checkpoints) {
        std::array<void *, 2 * kTrace> table{};
        for (int k = 0; k < kTrace; ++k) {   // large tensors: an allocation each, so that a user can drop them one by one
            const int64_t width = k < 4 ? 4 * H : H;
            values.push_back(emptyLike(p.x, {T, B, width}));
            clamped.push_back(emptyLike(p.x, {T, B, width}, at::kByte));
            table[k] = pointer<void>(values.back());
            table[kTrace + k] = pointer<void>(clamped.back());
        }
        std::memcpy(&trace, table.data(), sizeof(trace));
        const int64_t bias = p.bIh.defined() ? 4 * H : 0;
        const std::vector<Shape> shapes{p.wIh.sizes().vec(), p.wHh.sizes().vec(), {bias}, {bias}, {1, B, H}, {1, B, H}};
        masters.push_back(emptyLike(p.x, p.x.sizes()));
        masterClamped.push_back(emptyLike(p.x, p.x.sizes(), at::kBool));
        for (Tensor &t : carve(p.x, at::kFloat, shapes)) masters.push_back(std::move(t));
        for (Tensor &t : carve(p.x, at::kBool, shapes)) masterClamped.push_back(std::move(t));   // every flag is written
        for (int k = 0; k < kMasters; ++k) {
            table[k] = pointer<void>(masters[k]);
            table[kMasters + k] = pointer<void>(masterClamped[k]);
        }
        std::memcpy(&saved, table.data(), sizeof(saved));
    }
    const Tensor ws = emptyLike(p.x, {static_cast<int64_t>(rxmet_lstm_workspace_bytes(1, p.T, p.B, p.I, p.H))}, at::kByte);
    int status;
    {
        const pybind11::gil_scoped_release release;
        status = rxmet_lstm_forward_quantized(
            p.T, p.B, p.I, p.H, pointer<float>(p.wIh), pointer<float>(p.wHh), pointer<float>(p.bIh), pointer<float>(p.bHh),
            pointer<float>(p.x), pointer<float>(p.h0), pointer<float>(p.c0), params, requireExact, pointer<float>(out),
            pointer<float>(hn), pointer<float>(cn), checkpoints ? &trace : nullptr, checkpoints ? &saved : nullptr, ws.data_ptr(),
            static_cast<size_t>(ws.numel()), streamOf(p.x));
    }
    return {status, out, hn, cn, std::move(values), std::move(clamped), std::move(masters), std::move(masterClamped)};
}

Tensor maskTensor(const Tensor &t, const char *name, at::IntArrayRef shape, const c10::Device &device, bool allowEmpty = false) {
    TORCH_CHECK(t.scalar_type() == at::kBool || t.scalar_type() == at::kByte, name, " must be a bool or uint8 tensor");
    TORCH_CHECK(t.device() == device, name, " is on another device");
    if (allowEmpty && t.numel() == 0) return Tensor();
    TORCH_CHECK(t.sizes() == shape, name, " shape mismatch");
    return t.contiguous();
}

std::pair<int, std::vector<Tensor>> lstmBackwardQat(const std::vector<Tensor> &masters, bool batchFirst, uintptr_t paramsAddress,
                                                    const std::vector<Tensor> &trace, const Tensor &gradOutput,
                                                    const Tensor &gradHidden, const Tensor &gradCell,
                                                    const std::vector<Tensor> &masterMasks, const std::vector<Tensor> &traceMasks) {
    const auto *params = reinterpret_cast<const rxmet_lstm_quant_params *>(paramsAddress);
    const bool bias = params->bias_enabled != 0;
    const LstmInputs p(masters[0], masters[1], masters[2], bias ? MaybeTensor(masters[3]) : MaybeTensor(),
                       bias ? MaybeTensor(masters[4]) : MaybeTensor(), masters[5], masters[6], batchFirst);
    const int64_t T = p.T, B = p.B, H = p.H, C = 4 * H;
    auto shaped = [](const Tensor &given, const char *name, at::IntArrayRef shape) {
        Tensor t = lstmFloat(given, name);
        TORCH_CHECK(t.sizes() == shape, name, " shape mismatch");
        return t;
    };
    const Tensor gates = shaped(trace[0], "gate_outputs", {T, B, C}), cells = shaped(trace[1], "cell_states", {T, B, H});
    const Tensor tanhs = shaped(trace[2], "cell_tanh_outputs", {T, B, H}), hiddens = shaped(trace[3], "hidden_outputs", {T, B, H});
    const Tensor gOut = shaped(gradOutput, "grad_output", {T, B, H}), gH = shaped(gradHidden, "grad_final_hidden", {B, H});
    const Tensor gC = shaped(gradCell, "grad_final_cell", {B, H});
    TORCH_CHECK(masterMasks.empty() == traceMasks.empty(), "master_masks and checkpoint_masks must be given together");
    rxmet_lstm_backward_masks flags{};
    static_assert(sizeof(flags) == (kMasters + kTrace) * sizeof(void *), "pointer table");
    std::vector<Tensor> keep;
    const c10::Device device = p.x.device();
    const c10::cuda::CUDAGuard guard(device);
    if (!masterMasks.empty()) {
        TORCH_CHECK(masterMasks.size() == kMasters && traceMasks.size() == kTrace,
                    "master_masks and checkpoint_masks must hold 7 tensors each");
        const char *const traceNames[] = {"weight_ih_linear_mask", "weight_hh_linear_mask", "gate_inputs_mask", "gate_outputs_mask",
                                          "cell_states_mask", "cell_tanh_outputs_mask", "hidden_outputs_mask"};
        Tensor first = maskTensor(masterMasks[0], "input_mask", masters[0].sizes(), device);
        keep.push_back(batchFirst ? first.transpose(0, 1).contiguous() : first);
        keep.push_back(maskTensor(masterMasks[1], "weight_ih_mask", p.wIh.sizes(), device));
        keep.push_back(maskTensor(masterMasks[2], "weight_hh_mask", p.wHh.sizes(), device));
        keep.push_back(maskTensor(masterMasks[3], "bias_ih_mask", {C}, device, true));
        keep.push_back(maskTensor(masterMasks[4], "bias_hh_mask", {C}, device, true));
        keep.push_back(maskTensor(masterMasks[5], "initial_hidden_mask", {1, B, H}, device));
        keep.push_back(maskTensor(masterMasks[6], "initial_cell_mask", {1, B, H}, device));
        for (int k = 0; k < kTrace; ++k) keep.push_back(maskTensor(traceMasks[k], traceNames[k], {T, B, k < 4 ? C : H}, device));
        std::array<void *, kMasters + kTrace> table;
        for (size_t k = 0; k < table.size(); ++k) table[k] = keep[k].defined() ? keep[k].data_ptr() : nullptr;
        std::memcpy(&flags, table.data(), sizeof(flags));
    }
    std::vector<Tensor> grads{emptyLike(p.x, {T, B, p.I})};
    for (Tensor &t : carve(p.x, at::kFloat, {p.wIh.sizes().vec(), p.wHh.sizes().vec(), {C}, {C}, {B, H}, {B, H}}))
        grads.push_back(std::move(t));
    rxmet_lstm_gradients out{};
    static_assert(sizeof(out) == kMasters * sizeof(void *), "pointer table");
    std::array<void *, kMasters> table;
    for (int k = 0; k < kMasters; ++k) table[k] = grads[k].data_ptr();
    std::memcpy(&out, table.data(), sizeof(out));
    const auto *bits = params->config.bitwidth;
    const bool tensorCores = bits[RXMET_LSTM_WEIGHT_IH] <= 8 && bits[RXMET_LSTM_WEIGHT_HH] <= 8 && bits[RXMET_LSTM_INPUT] <= 16 &&
                             bits[RXMET_LSTM_OUTPUT] <= 16;
    const Tensor ws = emptyLike(p.x, {static_cast<int64_t>(rxmet_lstm_workspace_bytes(tensorCores ? 2 : 4, p.T, p.B, p.I, p.H))}, at::kByte);
    int status;
    {
        const pybind11::gil_scoped_release release;
        status = rxmet_lstm_backward_qat(
            p.T, p.B, p.I, p.H, params, pointer<float>(p.wIh), pointer<float>(p.wHh), pointer<float>(p.x), pointer<float>(p.h0),
            pointer<float>(p.c0), pointer<float>(gates), pointer<float>(cells), pointer<float>(tanhs), pointer<float>(hiddens),
            pointer<float>(gOut), pointer<float>(gH), pointer<float>(gC), masterMasks.empty() ? nullptr : &flags, &out,
            ws.data_ptr(), static_cast<size_t>(ws.numel()), streamOf(p.x));
    }
    if (batchFirst) grads[0] = grads[0].transpose(0, 1);
    return {status, std::move(grads)};
}

// ---- learned-grid quantize-dequantize -----------------------------------------------------------------------------

void checkStatus(int status, const char *what) {
    if (status == RXMET_OK) return;
    const std::string message = std::string(what) + ": " + rxmet_last_error();
    if (status == RXMET_ERR_INVALID_ARGUMENT) throw pybind11::value_error(message);
    TORCH_CHECK(false, message, " (status ", status, ")");
}

Tensor gridValues(const Tensor &t) { return (t.scalar_type() == at::kFloat ? t : t.to(at::kFloat)).contiguous(); }

// Saves the input itself instead of a mask: the backward recomputes the flags in the pass that reads it anyway.
struct QuantDequant : torch::autograd::Function<QuantDequant> {
    static Tensor forward(torch::autograd::AutogradContext *ctx, const Tensor &tensor, const Tensor &scale, const Tensor &offset,
                          int64_t qmin, int64_t qmax, bool reciprocal, int64_t outer, int64_t channels, int64_t inner) {
        const c10::cuda::CUDAGuard guard(tensor.device());   // launch on the tensor's device, whatever device is current
        const Tensor x = tensor.contiguous(), s = gridValues(scale), o = gridValues(offset);
        Tensor y = at::empty_like(x);
        checkStatus(rxmet_affine_qdq_forward(x.const_data_ptr<float>(), outer, channels, inner, s.const_data_ptr<float>(),
                                          o.const_data_ptr<float>(), static_cast<int>(qmin), static_cast<int>(qmax), reciprocal,
                                          y.mutable_data_ptr<float>(), nullptr, streamOf(x)),
                 "affine_qdq.forward");
        ctx->save_for_backward({tensor, scale, offset});
        ctx->saved_data["plan"] = std::vector<int64_t>{qmin, qmax, reciprocal, outer, channels, inner};
        return y;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const auto plan = ctx->saved_data["plan"].toIntVector();
        const uint64_t outer = plan[3], channels = plan[4], inner = plan[5];
        torch::autograd::variable_list out(9);
        if (!grads[0].defined()) return out;
        const at::NoGradGuard noGrad;
        const c10::cuda::CUDAGuard guard(saved[0].device());
        const Tensor x = saved[0].contiguous(), s = gridValues(saved[1]), o = gridValues(saved[2]), g = gridValues(grads[0]);
        const bool wantScale = ctx->needs_input_grad(1), wantOffset = ctx->needs_input_grad(2);
        Tensor ws;
        size_t bytes = 0;
        if (ctx->needs_input_grad(0)) out[0] = at::empty_like(x);
        if (wantScale) out[1] = emptyLike(x, saved[1].sizes());
        if (wantOffset) out[2] = emptyLike(x, saved[2].sizes());
        if (wantScale || wantOffset) {
            bytes = rxmet_affine_qdq_backward_workspace_bytes(outer, channels, inner);
            if (bytes > 0) ws = emptyLike(x, {static_cast<int64_t>(bytes)}, at::kByte);
        }
        auto raw = [](const Tensor &t) { return t.defined() ? static_cast<float *>(t.data_ptr()) : nullptr; };
        checkStatus(rxmet_affine_qdq_backward(raw(g), raw(x), outer, channels, inner, raw(s), raw(o), static_cast<int>(plan[0]),
                                           static_cast<int>(plan[1]), static_cast<int>(plan[2]), raw(out[0]), raw(out[1]),
                                           raw(out[2]), ws.defined() ? ws.data_ptr() : nullptr, bytes, streamOf(x)),
                 "affine_qdq.backward");
        return out;
    }
};

Tensor quantizeDequantize(const Tensor &tensor, const Tensor &scale, const Tensor &offset, int64_t qmin, int64_t qmax,
                          bool reciprocal, int64_t outer, int64_t channels, int64_t inner) {
    return QuantDequant::apply(tensor, scale, offset, qmin, qmax, reciprocal, outer, channels, inner);
}

// ---- token mixer: residual norm, product of codes, linear attention with decays ---------------------------------------------

int typeOf(const Tensor &t, const char *name) {
    if (t.scalar_type() == at::kFloat) return RXMET_TYPE_F32;
    if (t.scalar_type() == at::kBFloat16) return RXMET_TYPE_BF16;
    TORCH_CHECK(t.scalar_type() == at::kHalf, name, " must be a float32, bfloat16 or float16 tensor");
    return RXMET_TYPE_F16;
}

void sameDevice(const Tensor &t, const Tensor &like, const char *name) {
    TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be a CUDA tensor on ", like.device());
}

// Sizes that the C ABI takes in 32 bits, refused before they are cut and before anything is copied.
void checkSizes(at::IntArrayRef sizes, const char *what) {
    for (const int64_t n : sizes) TORCH_CHECK(n <= INT32_MAX, what, ": a size of ", n, ", at most ", INT32_MAX);
}

// [rows][width] with neighbouring elements, a view where the strides allow one; the distance of its rows.
Tensor asRows(const Tensor &t) {
    if (t.dim() == 2 && t.stride(1) == 1) return t;
    const Tensor flat = t.reshape({t.numel() / t.size(-1), t.size(-1)});
    return flat.stride(1) == 1 || flat.size(1) == 1 ? flat : flat.contiguous();
}
int64_t pitchOf(const Tensor &rows) { return rows.size(0) > 1 ? rows.stride(0) : rows.size(1); }

// Codes of rows that start on 16 bytes, as the products read them; the padding is not part of the tensor and holds nothing.
Tensor emptyCodes(const Tensor &like, at::IntArrayRef shape) {
    const int64_t width = shape.back(), pitch = (width + 15) / 16 * 16;
    Shape padded = shape.vec();
    padded.back() = pitch;
    const Tensor held = emptyLike(like, padded, at::kChar);
    return pitch == width ? held : held.narrow(-1, 0, width);
}

struct NormArguments {
    Tensor x, residual, weight;
    int type, weightType;
    int64_t rows, width;
    NormArguments(const Tensor &input, const MaybeTensor &added, const MaybeTensor &weights, const char *what) {
        TORCH_CHECK(input.is_cuda() && input.dim() >= 1 && input.size(-1) > 0, what, ": x must be a CUDA tensor with a last dimension");
        checkSizes({input.size(-1)}, what);
        type = typeOf(input, "x");
        width = input.size(-1);
        x = asRows(input);
        rows = x.size(0);
        if (added) {
            sameDevice(*added, input, "residual");
            TORCH_CHECK(added->sizes() == input.sizes() && added->scalar_type() == input.scalar_type(), what,
                        ": residual must have the shape and type of x");
            residual = asRows(*added);
        }
        weightType = type;
        if (weights) {
            sameDevice(*weights, input, "weight");
            weightType = typeOf(*weights, "weight");
            TORCH_CHECK(weights->dim() == 1 && weights->size(0) == width, what, ": weight must have shape [", width, "]");
            weight = weights->contiguous();
        }
    }
};

const void *dataOf(const Tensor &t) { return t.defined() && t.numel() > 0 ? t.const_data_ptr() : nullptr; }
void *mutableOf(const Tensor &t) { return t.defined() && t.numel() > 0 ? t.mutable_data_ptr() : nullptr; }

// Gradients that are to be differentiated again (create_graph) fail when they are: as constants they would leave their terms out in silence.  `from`: the tensors that they
// depend on, to which the failing node is linked, since only nodes on a way to what is asked for run.
torch::autograd::variable_list differentiatedOnce(torch::autograd::variable_list grads, torch::autograd::variable_list from, const char *what) {
    torch::autograd::variable_list all;
    for (const Tensor &g : grads)
        if (g.defined()) all.push_back(g.detach());
    const size_t count = all.size();
    for (Tensor &t : from)
        if (t.defined() && t.requires_grad()) all.push_back(std::move(t));
    if (count == 0 || all.size() == count) return grads;
    const auto node = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " has no second derivatives", static_cast<int64_t>(all.size()));
    const auto linked = (*node)(std::move(all));
    size_t i = 0;
    for (Tensor &g : grads)
        if (g.defined()) g = linked[i++];
    return grads;
}

// The outputs are y and, with a residual, total.
struct AddRmsNorm : torch::autograd::Function<AddRmsNorm> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const Tensor &x, const Tensor &weight,
                                                  const MaybeTensor &residual, double eps) {
        const NormArguments a(x, residual, weight, "add_rms_norm");
        const c10::cuda::CUDAGuard guard(x.device());
        Tensor y = emptyLike(x, x.sizes(), x.scalar_type()), total;
        if (residual) total = emptyLike(x, x.sizes(), x.scalar_type());
        const Tensor rms = emptyLike(x, {a.rows});
        checkStatus(rxmet_add_rms_norm(a.rows, static_cast<int>(a.width), a.type, dataOf(a.x), pitchOf(a.x), dataOf(a.residual),
                                       residual ? pitchOf(a.residual) : 0, dataOf(a.weight), a.weightType, static_cast<float>(eps),
                                       mutableOf(total), mutableOf(y), pointer<float>(rms), streamOf(x)),
                    "add_rms_norm");
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({x, rms, weight, residual ? *residual : Tensor()});
        if (residual) return {y, total};
        return {y};
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
        if (!at::GradMode::is_enabled()) return gradients(ctx, std::move(grads));
        auto from = ctx->get_saved_variables();
        from.insert(from.end(), grads.begin(), grads.end());
        return differentiatedOnce(gradients(ctx, std::move(grads)), std::move(from), "add_rms_norm");
    }

    static torch::autograd::variable_list gradients(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        torch::autograd::variable_list out(4);
        const at::NoGradGuard noGrad;
        const Tensor given = saved[0], rms = saved[1], weight = saved[2].contiguous();
        const c10::cuda::CUDAGuard guard(given.device());
        const Tensor dtotal = grads.size() > 1 && grads[1].defined() ? grads[1].contiguous() : Tensor();
        if (!grads[0].defined()) {
            if (dtotal.defined()) out[0] = out[2] = dtotal;
            return out;
        }
        const Tensor dy = grads[0].contiguous(), x = asRows(given), residual = saved[3].defined() ? asRows(saved[3]) : Tensor();
        const int type = typeOf(given, "x"), weightType = typeOf(weight, "weight"), width = static_cast<int>(given.size(-1));
        const Tensor dx = emptyLike(given, given.sizes(), given.scalar_type());
        Tensor ws;
        size_t bytes = 0;
        if (ctx->needs_input_grad(1)) {
            out[1] = emptyLike(given, {width}, weight.scalar_type());
            bytes = rxmet_add_rms_norm_backward_workspace_bytes(x.size(0), width, type);
            ws = emptyLike(given, {static_cast<int64_t>(bytes)}, at::kByte);
        }
        checkStatus(rxmet_add_rms_norm_backward(x.size(0), width, type, dataOf(dy), dataOf(dtotal), dataOf(x), pitchOf(x), dataOf(residual),
                                                residual.defined() ? pitchOf(residual) : 0, pointer<float>(rms),
                                                dataOf(weight), weightType, mutableOf(dx), mutableOf(out[1]), mutableOf(ws), bytes, streamOf(given)),
                    "add_rms_norm backward");
        out[0] = dx;
        if (saved[3].defined() && ctx->needs_input_grad(2)) out[2] = dx;   // an absent residual has no place of its own
        return out;
    }
};

// A trace would record the buffer that an output is written to, and not the kernel that writes it.
void refuseTrace(const char *what) { TORCH_CHECK(!torch::jit::tracer::isTracing(), what, " cannot be traced: the traced function would return memory that nothing writes"); }

std::vector<Tensor> addRmsNorm(const Tensor &x, const Tensor &weight, const MaybeTensor &residual, double eps) {
    refuseTrace("add_rms_norm");
    return AddRmsNorm::apply(x, weight, residual, eps);
}

// Codes, scales and (with a residual) total.
std::vector<Tensor> addRmsNormCodes(const Tensor &x, const MaybeTensor &weight, const MaybeTensor &residual, double eps) {
    refuseTrace("add_rms_norm_codes");
    const NormArguments a(x, residual, weight, "add_rms_norm_codes");
    const c10::cuda::CUDAGuard guard(x.device());
    std::vector<Tensor> out{emptyCodes(x, x.sizes()), emptyLike(x, x.sizes().slice(0, x.dim() - 1))};
    if (residual) out.push_back(emptyLike(x, x.sizes(), x.scalar_type()));
    checkStatus(rxmet_add_rms_norm_codes(a.rows, static_cast<int>(a.width), a.type, dataOf(a.x), pitchOf(a.x), dataOf(a.residual),
                                         residual ? pitchOf(a.residual) : 0, dataOf(a.weight), a.weightType, static_cast<float>(eps),
                                         residual ? mutableOf(out[2]) : nullptr, static_cast<int8_t *>(mutableOf(out[0])), (a.width + 15) / 16 * 16,
                                         pointer<float>(out[1]), streamOf(x)),
                "add_rms_norm_codes");
    return out;
}

Tensor codedLinear(const Tensor &codes, const Tensor &scale, const Tensor &weight, const Tensor &weightScale, const MaybeTensor &bias,
                   int activation, const MaybeTensor &residual, int outType) {
    refuseTrace("coded_linear");
    constexpr at::ScalarType kTypes[] = {at::kFloat, at::kBFloat16, at::kHalf};
    TORCH_CHECK(outType >= 0 && outType <= 2, "coded_linear: unknown output type");
    TORCH_CHECK(codes.is_cuda() && codes.scalar_type() == at::kChar && codes.dim() >= 1, "codes must be a CUDA int8 tensor");
    sameDevice(weight, codes, "weight codes");
    TORCH_CHECK(weight.scalar_type() == at::kChar && weight.dim() == 2, "weight codes must be an int8 tensor of two dimensions");
    checkSizes(weight.sizes(), "coded_linear");
    const int64_t inner = weight.size(1), outer = weight.size(0);
    TORCH_CHECK(inner > 0 && outer > 0 && codes.size(-1) == inner, "coded_linear: codes of ", codes.size(-1), " elements for a weight of shape ", listText(weight.sizes()));
    sameDevice(scale, codes, "scale");
    TORCH_CHECK(scale.scalar_type() == at::kFloat && scale.sizes() == codes.sizes().slice(0, codes.dim() - 1), "scale must be float32 with the shape of codes but its last dimension");
    sameDevice(weightScale, codes, "weight scale");
    TORCH_CHECK(weightScale.scalar_type() == at::kFloat && weightScale.dim() == 1 && weightScale.size(0) == outer, "weight scale must be float32 of shape [", outer, "]");
    Shape shape = codes.sizes().vec();
    shape.back() = outer;
    const c10::cuda::CUDAGuard guard(codes.device());
    // rows that share memory (a view that repeats one) are laid out apart: the C ABI takes none that overlap
    auto rowsApart = [](const Tensor &t) {
        const Tensor r = asRows(t);
        return r.size(0) > 1 && r.stride(0) < r.size(1) ? r.contiguous() : r;
    };
    const Tensor rows = rowsApart(codes), weights = rowsApart(weight), scales = scale.contiguous(), weightScales = weightScale.contiguous();
    Tensor added, biases;
    if (bias) {
        sameDevice(*bias, codes, "bias");
        TORCH_CHECK(bias->scalar_type() == at::kFloat && bias->dim() == 1 && bias->size(0) == outer, "bias must be float32 of shape [", outer, "]");
        biases = bias->contiguous();
    }
    if (residual) {
        sameDevice(*residual, codes, "residual");
        TORCH_CHECK(residual->scalar_type() == kTypes[outType] && residual->sizes() == at::IntArrayRef(shape), "residual must have the type and shape of the output, ", listText(shape));
        added = asRows(*residual);
    }
    const Tensor out = emptyLike(codes, shape, kTypes[outType]);
    checkStatus(rxmet_coded_linear(rows.size(0), static_cast<int>(inner), static_cast<int>(outer), static_cast<const int8_t *>(dataOf(rows)), pitchOf(rows),
                                   pointer<float>(scales), static_cast<const int8_t *>(dataOf(weights)), pitchOf(weights), pointer<float>(weightScales),
                                   pointer<float>(biases), activation, dataOf(added), residual ? pitchOf(added) : 0, outType, mutableOf(out), streamOf(codes)),
                "coded_linear");
    return out;
}

// Arguments of linear attention as the C ABI takes them; tensors of three dimensions are single tokens.
struct AttentionArguments {
    Tensor q, k, v, logDecay, lengths, state;
    rxmet_decayed_attention problem{};
    Shape stateShape;

    static rxmet_head_tensor view(const Tensor &t) {
        const bool step = t.dim() == 3;
        return {dataOf(t), t.stride(0), step ? 0 : t.stride(1), t.stride(step ? 1 : 2), static_cast<int32_t>(t.size(step ? 1 : 2))};
    }
    // Neighbouring elements of a head; sequences of 16-bit elements also start every head, token and row on 16 bytes, as TMA copies them (a copy where
    // they do not: the kernel without TMA takes several times as long).
    static Tensor rowsOf(const Tensor &t) {
        if (t.dim() == 4 && t.scalar_type() != at::kFloat && t.size(1) >= 32) {
            bool fits = (t.stride(3) == 1 || t.size(3) == 1) && reinterpret_cast<uintptr_t>(dataOf(t)) % 16 == 0;
            for (int i = 0; i < 3; ++i) fits = fits && (t.size(i) == 1 || (t.stride(i) > 0 && t.stride(i) % 8 == 0));
            if (fits) return t;
            const Tensor copy = emptyLike(t, {t.size(0), t.size(1), t.size(2), (t.size(3) + 7) / 8 * 8}, t.scalar_type()).narrow(3, 0, t.size(3));
            copy.copy_(t);
            return copy;
        }
        return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous();
    }

    AttentionArguments(const Tensor &queries, const Tensor &keys, const Tensor &values, const Tensor &decays, const MaybeTensor &start,
                       const MaybeTensor &counts, double scale, int64_t dims) {
        TORCH_CHECK(queries.is_cuda() && queries.dim() == dims, "q must be a CUDA tensor of ", dims, " dimensions");
        problem.type = typeOf(queries, "q");
        for (const Tensor *t : {&queries, &keys, &values, &decays}) checkSizes(t->sizes(), "decayed_attention");
        for (const auto &[t, name] : {std::pair<const Tensor &, const char *>{keys, "k"}, {values, "v"}}) {
            sameDevice(t, queries, name);
            TORCH_CHECK(t.dim() == dims && t.scalar_type() == queries.scalar_type(), name, " must have the dimensions and type of q");
            for (int64_t i = 0; i < dims - 2; ++i) TORCH_CHECK(t.size(i) == queries.size(i), name, " must have batch and tokens of q");
        }
        TORCH_CHECK(keys.size(-1) == queries.size(-1), "q and k must have heads of one size");
        sameDevice(decays, queries, "log_decay");
        TORCH_CHECK(decays.scalar_type() == at::kFloat && decays.dim() == 1 && decays.size(0) > 0, "log_decay must be a float32 tensor of one dimension, the heads");
        q = rowsOf(queries);
        k = rowsOf(keys);
        v = rowsOf(values);
        logDecay = decays.contiguous();
        problem.batch = static_cast<int32_t>(q.size(0));
        problem.tokens = dims == 3 ? 1 : static_cast<int32_t>(q.size(1));
        problem.heads = static_cast<int32_t>(logDecay.size(0));
        problem.key_dim = static_cast<int32_t>(q.size(-1));
        problem.value_dim = static_cast<int32_t>(v.size(-1));
        stateShape = {problem.batch, problem.heads, problem.key_dim, problem.value_dim};
        if (start) state = checkedState(*start, "state").contiguous();
        if (counts) {
            sameDevice(*counts, queries, "lengths");
            TORCH_CHECK(counts->dim() == 1 && counts->size(0) == problem.batch && at::isIntegralType(counts->scalar_type(), true), "lengths must be integers of shape [", problem.batch, "]");
            // of 64 bits, they are cut to the tokens that there are before they are cut to 32
            const int64_t most = dims == 3 ? 1 : queries.size(1);
            lengths = (counts->scalar_type() == at::kLong ? at::clamp(*counts, 0, most) : *counts).to(at::kInt).contiguous();
        }
        problem.q = view(q);
        problem.k = view(k);
        problem.v = view(v);
        problem.log_decay = logDecay.const_data_ptr<float>();
        problem.lengths = lengths.defined() ? lengths.const_data_ptr<int32_t>() : nullptr;
        problem.scale = static_cast<float>(scale);
    }
    const Tensor &checkedState(const Tensor &t, const char *name) const {
        sameDevice(t, q, name);
        TORCH_CHECK(t.scalar_type() == at::kFloat && t.sizes() == at::IntArrayRef(stateShape), name, " must be float32 of shape ", listText(stateShape));
        return t;
    }
    Tensor workspaceFor(bool backward, size_t &bytes) const {
        bytes = rxmet_decayed_attention_workspace_bytes(&problem, backward);
        return bytes > 0 ? emptyLike(q, {static_cast<int64_t>(bytes)}, at::kByte) : Tensor();
    }
    void forward(const Tensor &out, const Tensor &last) const {
        size_t bytes;
        const Tensor ws = workspaceFor(false, bytes);
        checkStatus(rxmet_decayed_attention_forward(&problem, pointer<float>(state), mutableOf(out), pointer<float>(last), mutableOf(ws), bytes, streamOf(q)), "decayed_attention");
    }
};

struct DecayedAttention : torch::autograd::Function<DecayedAttention> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &logDecay,
                                                  const MaybeTensor &state, const MaybeTensor &lengths, double scale) {
        const AttentionArguments a(q, k, v, logDecay, state, lengths, scale, 4);
        const c10::cuda::CUDAGuard guard(q.device());
        const Tensor out = emptyLike(q, {q.size(0), q.size(1), logDecay.size(0), v.size(3)}, q.scalar_type()), last = emptyLike(q, a.stateShape);
        a.forward(out, last);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({q, k, v, a.logDecay, state ? *state : Tensor(), a.lengths});
        ctx->saved_data["scale"] = scale;
        return {out, last};
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
        if (!at::GradMode::is_enabled()) return gradients(ctx, std::move(grads));
        auto from = ctx->get_saved_variables();
        from.insert(from.end(), grads.begin(), grads.end());
        return differentiatedOnce(gradients(ctx, std::move(grads)), std::move(from), "decayed_attention");
    }

    static torch::autograd::variable_list gradients(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        torch::autograd::variable_list out(7);
        if (!grads[0].defined() && !grads[1].defined()) return out;
        const at::NoGradGuard noGrad;
        auto maybe = [](const Tensor &t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); };
        const Tensor q = saved[0];
        const AttentionArguments a(q.detach(), saved[1].detach(), saved[2].detach(), saved[3], maybe(saved[4]), maybe(saved[5]), ctx->saved_data["scale"].toDouble(), 4);
        const c10::cuda::CUDAGuard guard(q.device());
        const Tensor dout = grads[0].defined() ? AttentionArguments::rowsOf(grads[0])
                                               : at::zeros({q.size(0), q.size(1), a.problem.heads, a.problem.value_dim}, q.options());
        const Tensor dlast = grads[1].defined() ? grads[1].contiguous() : Tensor();
        for (int i = 0; i < 3; ++i)
            if (ctx->needs_input_grad(i)) out[i] = emptyLike(q, saved[i].sizes(), q.scalar_type());
        if (saved[4].defined() && ctx->needs_input_grad(4)) out[4] = emptyLike(q, a.stateShape);
        size_t bytes;
        const Tensor ws = a.workspaceFor(true, bytes);
        const rxmet_head_tensor d = AttentionArguments::view(dout);
        checkStatus(rxmet_decayed_attention_backward(&a.problem, pointer<float>(a.state), &d, pointer<float>(dlast), mutableOf(out[0]), mutableOf(out[1]),
                                                     mutableOf(out[2]), pointer<float>(out[4]), mutableOf(ws), bytes, streamOf(q)),
                    "decayed_attention backward");
        return out;
    }
};

void constantDecay(const Tensor &decays) {
    TORCH_CHECK(!at::GradMode::is_enabled() || !decays.requires_grad(), "log_decay is a constant of the layer: it has no gradient");
}

std::vector<Tensor> decayedAttention(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &logDecay, const MaybeTensor &state,
                                     const MaybeTensor &lengths, double scale) {
    refuseTrace("decayed_attention");
    constantDecay(logDecay);
    return DecayedAttention::apply(q, k, v, logDecay, state, lengths, scale);
}

// One token for each row; the states go to `newState`, which may be `state` itself.
Tensor decayedAttentionStep(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &logDecay, const Tensor &state, const Tensor &newState,
                            const MaybeTensor &active, double scale) {
    refuseTrace("decayed_attention_step");
    constantDecay(logDecay);
    if (at::GradMode::is_enabled())
        for (const Tensor *t : {&q, &k, &v, &state, &newState})
            TORCH_CHECK(!t->requires_grad(), "decayed_attention_step has no gradient: use decayed_attention, or no_grad");
    const AttentionArguments a(q, k, v, logDecay, state, active, scale, 3);
    a.checkedState(newState, "new_state");
    TORCH_CHECK(newState.is_contiguous(), "new_state must be contiguous");
    const c10::cuda::CUDAGuard guard(q.device());
    const Tensor out = emptyLike(q, {q.size(0), logDecay.size(0), v.size(2)}, q.scalar_type());
    a.forward(out, newState);
    newState.unsafeGetTensorImpl()->bump_version();
    return out;
}

}  // namespace

PYBIND11_MODULE(_binding, m) {
    m.def("workspace", [](int device, int64_t bytes) { return workspace(c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(device)), bytes); });
    m.def("gru_forward_quant", &gruForwardQuant);
    m.def("gru_backward_quant", &gruBackwardQuant);
    m.def("lstm_forward_quant", &lstmForwardQuant);
    m.def("lstm_backward_qat", &lstmBackwardQat);
    m.def("add_rms_norm", &addRmsNorm, pybind11::call_guard<pybind11::gil_scoped_release>());
    m.def("add_rms_norm_codes", &addRmsNormCodes, pybind11::call_guard<pybind11::gil_scoped_release>());
    m.def("coded_linear", &codedLinear, pybind11::call_guard<pybind11::gil_scoped_release>());
    m.def("decayed_attention", &decayedAttention, pybind11::call_guard<pybind11::gil_scoped_release>());
    m.def("decayed_attention_step", &decayedAttentionStep, pybind11::call_guard<pybind11::gil_scoped_release>());
    m.def("quantize_dequantize", &quantizeDequantize, pybind11::call_guard<pybind11::gil_scoped_release>());
}
