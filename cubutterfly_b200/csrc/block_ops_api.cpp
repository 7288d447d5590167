// block_ops_api.cpp -- C entry points of the block norm and the gated linear
// recurrence: argument checks, then launches.  Nothing here allocates device
// memory, copies or synchronises.
#include <cmath>
#include <stdexcept>
#include <string>

#include <cubutterfly/cubutterfly_b200.h>

#include "block_ops.hpp"

namespace cubf {
void set_last_error(const std::string& message);
}

namespace {

using cubf::BlockType;

struct NotSupported : std::runtime_error {
    using std::runtime_error::runtime_error;
};

void require(bool ok, const char* what) {
    if (!ok) throw std::invalid_argument(what);
}
void supported(bool ok, const char* what) {
    if (!ok) throw NotSupported(what);
}
void check(cudaError_t e, const char* what) {
    if (e != cudaSuccess) throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(e));
}

// No exception leaves a C entry, one from keeping the message included.
cubutterflyStatus_t failed(cubutterflyStatus_t status, const char* message) noexcept {
    try {
        cubf::set_last_error(message);
    } catch (...) {
    }
    return status;
}

template <typename Body>
cubutterflyStatus_t guarded(Body&& body) noexcept {
    try {
        cubf::set_last_error("");
        body();
        return CUBUTTERFLY_STATUS_SUCCESS;
    } catch (const std::invalid_argument& e) {
        return failed(CUBUTTERFLY_STATUS_INVALID_VALUE, e.what());
    } catch (const NotSupported& e) {
        return failed(CUBUTTERFLY_STATUS_NOT_SUPPORTED, e.what());
    } catch (const std::exception& e) {
        return failed(CUBUTTERFLY_STATUS_CUDA_ERROR, e.what());
    } catch (...) {
        return failed(CUBUTTERFLY_STATUS_INTERNAL_ERROR, "unknown exception");
    }
}

BlockType type_of(int data_type, const char* what) {
    switch (data_type) {
        case CUBUTTERFLY_DATA_FP16: return BlockType::kF16;
        case CUBUTTERFLY_DATA_BF16: return BlockType::kBF16;
        case CUBUTTERFLY_DATA_FP32: return BlockType::kF32;
        default: throw NotSupported(std::string(what) + " must be FP16, BF16 or FP32");
    }
}

size_t element(BlockType t) { return t == BlockType::kF32 ? 4 : 2; }

bool element_aligned(const void* p, size_t size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }

// (FP32 or the block's type) -> is fp32
bool vector_is_32(const void* p, int type, BlockType block, const char* what) {
    if (!p) return false;
    const BlockType t = type_of(type, what);
    if (t != block && t != BlockType::kF32) throw NotSupported(std::string(what) + " must be the block's type or FP32");
    if (!element_aligned(p, element(t))) throw std::invalid_argument(std::string(what) + ": misaligned vector");
    return t == BlockType::kF32;
}

// ---- block norm ---------------------------------------------------------------------------------
size_t gate_groups(const cubutterflyB200BlockNorm_t& a) {
    return a.gate_rows > 1 && a.gate_rows < a.rows ? a.gate_rows : 1;
}

void check_norm_sizes(const cubutterflyB200BlockNorm_t* a) {
    require(a != nullptr, "block norm: null arguments");
    require(a->struct_size == sizeof(*a), "block norm: struct_size does not match this library's");
    require(a->dim >= 1, "block norm: dim must be at least 1");
    supported(a->dim <= cubf::kBlockNormMaxDim, "block norm: dim is limited to 16384");
    supported(a->rows <= 0x7fffffffULL, "block norm: rows are limited to 2^31 - 1");
    require(a->gate_rows <= 1 || a->rows == 0 || (a->gate_rows <= a->rows && a->rows % a->gate_rows == 0),
            "block norm: gate_rows must be 0, 1 or a divisor of rows");
}

cubf::BlockNormArgs norm_args(const cubutterflyB200BlockNorm_t* a, bool backward, BlockType* block, bool* residual32) {
    check_norm_sizes(a);
    *block = type_of(a->data_type, "block norm data_type");
    const BlockType res = type_of(a->residual_type, "block norm residual_type");
    supported(res == *block || res == BlockType::kF32, "block norm: residual_type must be data_type or FP32");
    *residual32 = res == BlockType::kF32;
    require(a->activation >= 0 && a->activation <= 2, "block norm: unknown gate activation");
    require((a->flags & ~7) == 0, "block norm: unknown flags");
    require(std::isfinite(a->residual_scale), "block norm: residual_scale must be finite");
    require(std::isfinite(a->epsilon) && a->epsilon >= 0, "block norm: epsilon must be finite and not negative");
    const bool pre = a->flags & CUBUTTERFLY_B200_PRE_NORM, rotate = a->flags & CUBUTTERFLY_B200_ROTATE;
    const bool post = a->flags & CUBUTTERFLY_B200_POST_NORM;
    require(a->x != nullptr, "block norm: null x");
    require(a->y || (!post && !a->post_weight && a->gate_rows == 0),
            "block norm: a post norm, its weight and a gate need the block output y");
    require(!a->post_weight || post, "block norm: post_weight without POST_NORM");
    require(!a->pre_weight || pre, "block norm: pre_weight without PRE_NORM");
    require(!rotate || pre, "block norm: ROTATE without PRE_NORM");
    require((a->gate != nullptr) == (a->gate_rows > 0), "block norm: gate and gate_rows must be given together");
    supported(!rotate || (a->dim >= cubf::kBlockNormMinRotate && (a->dim & (a->dim - 1)) == 0),
              "block norm: ROTATE needs a power-of-two dim from 64 to 16384");
    require(a->x_row >= a->dim && (!a->y || a->y_row >= a->dim) && (a->gate_rows <= 1 || a->gate_row >= a->dim),
            "block norm: a row stride is below dim");
    const size_t es = element(*block), er = element(res);
    require(element_aligned(a->x, er) && element_aligned(a->y, es), "block norm: misaligned input");

    cubf::BlockNormArgs n{};
    n.x = a->x;
    n.y = a->y;
    n.gate = a->gate;
    n.pre = a->pre_weight;
    n.post = a->post_weight;
    n.scales = a->scale;
    // a row's place is one 32 x 32 bit product
    auto bytes = [](size_t elements, size_t size) {
        supported(elements <= 0xffffffffULL / size, "block norm: a row stride is limited to 4 GiB");
        return static_cast<uint32_t>(elements * size);
    };
    n.x_bytes = bytes(a->x_row, er);
    n.y_bytes = a->y ? bytes(a->y_row, es) : 0;
    n.gate_row = a->gate_rows > 1 ? a->gate_row : 0;
    n.gate_bytes = bytes(n.gate_row, es);
    n.rows = a->rows;
    n.dim = static_cast<int>(a->dim);
    n.act = a->activation;
    n.scale = static_cast<float>(a->residual_scale);
    n.eps = static_cast<float>(a->epsilon);
    n.rotate_scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(a->dim)));
    n.post_norm = post;
    n.rotate = rotate;
    require(element_aligned(a->post_rms, 4) && element_aligned(a->pre_rms, 4), "block norm: misaligned post_rms or pre_rms");
    n.pre32 = vector_is_32(a->pre_weight, a->pre_type, *block, "block norm pre_type");
    n.post32 = vector_is_32(a->post_weight, a->post_type, *block, "block norm post_type");
    n.scales32 = vector_is_32(a->scale, a->scale_type, *block, "block norm scale_type");
    const size_t groups = gate_groups(*a);
    n.rows_per_gate = a->rows / groups;
    if (a->gate_rows == 0) {
        n.gate_mode = cubf::kGateNone;
    } else if (a->gate_rows == 1) {
        n.gate_mode = cubf::kGateChannel;
    } else {
        n.gate_mode = a->gate_rows == a->rows ? cubf::kGateFull : cubf::kGateGroups;
    }
    if (n.gate_mode == cubf::kGateFull)
        require(element_aligned(a->gate, es), "block norm: misaligned gate");
    else
        n.gate32 = vector_is_32(a->gate, a->gate_type, *block, "block norm gate_type");
    n.parts_per_group = cubf::block_norm_parts(n.rows_per_gate, groups, n.dim);
    if (!backward) {
        require(!pre == !a->normed, "block norm: normed and PRE_NORM must be given together");
        require((a->post_rms != nullptr) == (a->pre_rms != nullptr), "block norm: post_rms and pre_rms go together");
        require(element_aligned(a->residual, er) && element_aligned(a->normed, es), "block norm: misaligned output");
        require(a->normed == nullptr || (a->normed != a->x && a->normed != a->y && a->normed != a->residual),
                "block norm: normed must not alias another tensor");
        require(a->residual != a->x || !a->x || a->x_row == a->dim, "block norm: an in-place residual needs x_row = dim");
        require(a->residual == nullptr || a->residual != a->y, "block norm: residual must not alias y");
        n.residual = a->residual;
        n.normed = a->normed;
        n.r_post = a->post_rms;
        n.r_pre = a->pre_rms;
        return n;
    }
    // the kernel that adds the parameter gradients has a CTA for 32 channels of each group
    supported((groups + 3) * ((a->dim + 31) / 32) <= 0x7fffffffULL, "block norm: too many gate groups");
    require(!a->d_normed || pre, "block norm: d_normed without PRE_NORM");
    require(a->d_x != nullptr && (a->d_y != nullptr) == (a->y != nullptr), "block norm: d_x and, with y, d_y are needed");
    require((a->d_gate != nullptr) == (a->gate != nullptr) &&
                (a->d_pre_weight != nullptr) == (a->pre_weight != nullptr) &&
                (a->d_post_weight != nullptr) == (a->post_weight != nullptr) &&
                (a->d_scale != nullptr) == (a->scale != nullptr),
            "block norm: every gate, weight and scale needs its gradient");
    require((!a->d_residual || a->d_residual_row >= a->dim) && (!a->d_normed || a->d_normed_row >= a->dim),
            "block norm: a gradient's row stride is below dim");
    require((!post || a->post_rms) && (!a->d_normed || a->pre_rms), "block norm: the forward's post_rms / pre_rms are needed");
    require(element_aligned(a->d_residual, er) && element_aligned(a->d_normed, es) && element_aligned(a->d_x, er) &&
                element_aligned(a->d_y, es),
            "block norm: misaligned gradient");
    auto vector_aligned = [&](const void* p, bool is32) { return element_aligned(p, is32 ? 4 : es); };
    require(vector_aligned(a->d_gate, n.gate32) && vector_aligned(a->d_pre_weight, n.pre32) &&
                vector_aligned(a->d_post_weight, n.post32) && vector_aligned(a->d_scale, n.scales32),
            "block norm: misaligned gradient of a gate, weight or scale");
    n.d_residual = a->d_residual;
    n.d_normed = a->d_normed;
    n.d_residual_bytes = a->d_residual ? bytes(a->d_residual_row, er) : 0;
    n.d_normed_bytes = a->d_normed ? bytes(a->d_normed_row, es) : 0;
    n.r_post = a->post_rms;
    n.r_pre = a->pre_rms;
    n.d_x = a->d_x;
    n.d_y = a->d_y;
    n.d_gate = a->d_gate;
    n.d_pre = a->d_pre_weight;
    n.d_post = a->d_post_weight;
    n.d_scale = a->d_scale;
    n.need_q = a->d_pre_weight != nullptr;
    n.need_z = a->d_scale != nullptr;
    n.need_p = a->d_post_weight != nullptr || n.gate_mode == cubf::kGateChannel || n.gate_mode == cubf::kGateGroups;
    return n;
}

size_t norm_workspace(const cubutterflyB200BlockNorm_t& a) {
    const size_t groups = gate_groups(a);
    const size_t parts = groups * static_cast<size_t>(cubf::block_norm_parts(a.rows / groups, groups, static_cast<int>(a.dim)));
    return (parts * 3 * a.dim * sizeof(float) + 15) / 16 * 16;
}

// ---- gated scan ---------------------------------------------------------------------------------
void check_scan_sizes(const cubutterflyB200GatedScan_t* a) {
    require(a != nullptr, "gated scan: null arguments");
    require(a->struct_size == sizeof(*a), "gated scan: struct_size does not match this library's");
    require(a->dim >= 1, "gated scan: dim must be at least 1");
    supported(a->dim <= (1u << 24), "gated scan: dim is limited to 2^24");
    supported(a->length <= cubf::kGatedScanMaxLength, "gated scan: length is limited to 2^30 tokens");
    supported(a->batch <= (1u << 24) && a->sequences <= (1u << 30), "gated scan: too many sequences");
    require(!a->offsets || (a->batch == 1 && a->sequences >= 1),
            "gated scan: a packed batch has batch = 1 and at least one sequence");
    require(a->offsets || a->sequences == 0, "gated scan: sequences without offsets");
}

void check_exponent(double exponent, const char* what) { require(std::isfinite(exponent) && exponent > 0, what); }

cubf::GatedScanArgs scan_args(const cubutterflyB200GatedScan_t* a, bool backward, BlockType* block) {
    check_scan_sizes(a);
    *block = type_of(a->data_type, "gated scan data_type");
    check_exponent(a->exponent, "gated scan: exponent must be finite and positive");
    const size_t es = element(*block);
    const bool tokens = a->batch > 0 && a->length > 0;
    if (tokens) {
        require(a->x && a->recurrence_gate && a->input_gate, "gated scan: null input");
        for (const void* p : {a->x, a->recurrence_gate, a->input_gate})
            require(element_aligned(p, es), "gated scan: misaligned input");
        require(a->length == 1 || (a->x_token >= a->dim && a->recurrence_token >= a->dim && a->input_token >= a->dim),
                "gated scan: a token stride is below dim");
    }
    require(a->decay != nullptr, "gated scan: null decay");
    for (const void* p : {static_cast<const void*>(a->decay), static_cast<const void*>(a->initial_state),
                          static_cast<const void*>(a->offsets), static_cast<const void*>(a->chunk_states),
                          static_cast<const void*>(a->final_state), static_cast<const void*>(a->d_final_state),
                          static_cast<const void*>(a->d_initial_state), static_cast<const void*>(a->d_decay)})
        require(element_aligned(p, 4), "gated scan: misaligned vector or state");
    cubf::GatedScanArgs s{};
    s.x = a->x;
    s.r = a->recurrence_gate;
    s.i = a->input_gate;
    s.x_batch = a->x_batch;
    s.x_token = a->x_token;
    s.r_batch = a->recurrence_batch;
    s.r_token = a->recurrence_token;
    s.i_batch = a->input_batch;
    s.i_token = a->input_token;
    s.decay = a->decay;
    s.initial = a->initial_state;
    s.offsets = a->offsets;
    s.chunk_states = a->chunk_states;
    s.batch = static_cast<int>(a->batch);
    s.length = static_cast<int>(a->length);
    s.dim = static_cast<int>(a->dim);
    s.sequences = static_cast<int>(a->sequences);
    s.exponent = static_cast<float>(a->exponent);
    if (!backward) {
        require((a->h && element_aligned(a->h, es)) || !tokens, "gated scan: null or misaligned h");
        require(a->final_state != nullptr || a->batch == 0, "gated scan: null final_state");
        require(!tokens || (a->h != a->x && a->h != a->recurrence_gate && a->h != a->input_gate),
                "gated scan: h must not alias an input");
        require(!a->initial_state || a->initial_state != a->final_state,
                "gated scan: final_state must not alias initial_state");
        s.h = a->h;
        s.last = a->final_state;
        return s;
    }
    if (tokens) {
        require(a->d_h && a->chunk_states, "gated scan: the backward needs d_h and the forward's chunk_states");
        require(a->d_x && a->d_recurrence_gate && a->d_input_gate, "gated scan: null gradient");
        for (const void* p : {a->d_h, static_cast<const void*>(a->d_x), static_cast<const void*>(a->d_recurrence_gate),
                              static_cast<const void*>(a->d_input_gate)})
            require(element_aligned(p, es), "gated scan: misaligned gradient");
        require(a->length == 1 || a->dh_token >= a->dim, "gated scan: the token stride of d_h is below dim");
    }
    require(a->d_decay != nullptr, "gated scan: null d_decay");
    s.d_h = a->d_h;
    s.dh_batch = a->dh_batch;
    s.dh_token = a->dh_token;
    s.d_last = a->d_final_state;
    s.d_x = a->d_x;
    s.d_r = a->d_recurrence_gate;
    s.d_i = a->d_input_gate;
    s.d_decay = a->d_decay;
    s.d_initial = a->d_initial_state;
    return s;
}

size_t scan_workspace(const cubutterflyB200GatedScan_t& a) {
    return (a.batch * a.dim * sizeof(float) + 15) / 16 * 16;
}

}  // namespace

extern "C" cubutterflyStatus_t cubutterflyB200BlockNormForward(const cubutterflyB200BlockNorm_t* args,
                                                              cudaStream_t stream) {
    return guarded([&] {
        BlockType block;
        bool residual32;
        const cubf::BlockNormArgs a = norm_args(args, false, &block, &residual32);
        if (a.rows == 0) return;
        check(cubf::launch_block_norm(block, residual32, a, stream), "block norm launch");
    });
}

extern "C" cubutterflyStatus_t cubutterflyB200BlockNormGetWorkspaceSize(const cubutterflyB200BlockNorm_t* args,
                                                                       size_t* bytes) {
    return guarded([&] {
        check_norm_sizes(args);
        require(bytes != nullptr, "block norm: null size");
        *bytes = args->rows == 0 ? 0 : norm_workspace(*args);
    });
}

extern "C" cubutterflyStatus_t cubutterflyB200BlockNormBackward(const cubutterflyB200BlockNorm_t* args,
                                                               cudaStream_t stream) {
    return guarded([&] {
        BlockType block;
        bool residual32;
        cubf::BlockNormArgs a = norm_args(args, true, &block, &residual32);
        supported(a.rows > 0, "block norm: the backward of zero rows is the caller's zeros");
        require(args->workspace && args->workspace_bytes >= norm_workspace(*args) && element_aligned(args->workspace, 16),
                "block norm: the backward needs a 16-byte aligned workspace of the queried size");
        a.partials = static_cast<float*>(args->workspace);
        check(cubf::launch_block_norm_backward(block, residual32, a, gate_groups(*args), stream),
              "block norm backward launch");
    });
}

extern "C" cubutterflyStatus_t cubutterflyB200GatedScanForward(const cubutterflyB200GatedScan_t* args,
                                                              cudaStream_t stream) {
    return guarded([&] {
        BlockType block;
        const cubf::GatedScanArgs a = scan_args(args, false, &block);
        supported(a.length > 0 || a.batch == 0, "gated scan: of zero tokens the final states are the initial ones");
        if (a.batch == 0) return;
        check(cubf::launch_gated_scan(block, a, false, stream), "gated scan launch");
    });
}

extern "C" cubutterflyStatus_t cubutterflyB200GatedScanGetWorkspaceSize(const cubutterflyB200GatedScan_t* args,
                                                                       size_t* bytes) {
    return guarded([&] {
        check_scan_sizes(args);
        require(bytes != nullptr, "gated scan: null size");
        *bytes = args->batch == 0 || args->length == 0 ? 0 : scan_workspace(*args);
    });
}

extern "C" cubutterflyStatus_t cubutterflyB200GatedScanBackward(const cubutterflyB200GatedScan_t* args,
                                                               cudaStream_t stream) {
    return guarded([&] {
        BlockType block;
        cubf::GatedScanArgs a = scan_args(args, true, &block);
        supported(a.length > 0 && a.batch > 0, "gated scan: the backward of zero tokens is the caller's zeros");
        require(args->workspace && args->workspace_bytes >= scan_workspace(*args) && element_aligned(args->workspace, 16),
                "gated scan: the backward needs a 16-byte aligned workspace of the queried size");
        a.partials = static_cast<float*>(args->workspace);
        check(cubf::launch_gated_scan(block, a, true, stream), "gated scan backward launch");
    });
}

extern "C" cubutterflyStatus_t cubutterflyB200GatedScanStep(const cubutterflyB200GatedScanStep_t* a,
                                                           cudaStream_t stream) {
    return guarded([&] {
        require(a != nullptr, "gated scan step: null arguments");
        require(a->struct_size == sizeof(*a), "gated scan step: struct_size does not match this library's");
        require(a->dim >= 1, "gated scan step: dim must be at least 1");
        supported(a->dim <= (1u << 24) && a->batch <= 0x7fffffffULL && a->pool <= 0x7fffffffULL,
                  "gated scan step: too many requests, slots or channels");
        check_exponent(a->exponent, "gated scan step: exponent must be finite and positive");
        const BlockType block = type_of(a->data_type, "gated scan step data_type");
        if (a->batch == 0) return;
        require(a->x && a->recurrence_gate && a->input_gate && a->decay && a->h, "gated scan step: null tensor");
        require((a->state && a->new_state) || a->pool == 0, "gated scan step: null state");
        require(a->slots || a->pool >= a->batch, "gated scan step: without slots the pool needs a row per request");
        require(a->batch == 1 || (a->x_row >= a->dim && a->recurrence_row >= a->dim && a->input_row >= a->dim),
                "gated scan step: a row stride is below dim");
        for (const void* p : {a->x, a->recurrence_gate, a->input_gate, static_cast<const void*>(a->h)})
            require(element_aligned(p, element(block)), "gated scan step: misaligned tensor");
        for (const void* p : {static_cast<const void*>(a->decay), static_cast<const void*>(a->state),
                              static_cast<const void*>(a->new_state), static_cast<const void*>(a->slots)})
            require(element_aligned(p, 4), "gated scan step: misaligned vector or state");
        // in place, or apart: between, a request would read a row that another one's step writes
        const uintptr_t from = reinterpret_cast<uintptr_t>(a->state), to = reinterpret_cast<uintptr_t>(a->new_state);
        const size_t bytes = a->pool * a->dim * sizeof(float);
        require(from == to || from + bytes <= to || to + bytes <= from,
                "gated scan step: new_state must be state or not overlap it");
        cubf::GatedStepArgs s{};
        s.x = a->x;
        s.r = a->recurrence_gate;
        s.i = a->input_gate;
        s.x_row = a->x_row;
        s.r_row = a->recurrence_row;
        s.i_row = a->input_row;
        s.decay = a->decay;
        s.state = a->state;
        s.new_state = a->new_state;
        s.slots = a->slots;
        s.h = a->h;
        s.batch = a->batch;
        s.pool = a->pool;
        s.dim = static_cast<int>(a->dim);
        s.exponent = static_cast<float>(a->exponent);
        check(cubf::launch_gated_scan_step(block, s, stream), "gated scan step launch");
    });
}
