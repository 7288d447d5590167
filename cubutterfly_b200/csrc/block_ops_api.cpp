// block_ops_api.cpp -- C entry points of the block norm, the gated linear
// recurrence, the gated delta rule and the norm of queries and keys: argument
// checks, then launches.  Nothing here allocates device
// memory, copies or synchronises.
#include <algorithm>
#include <cmath>
#include <stdexcept>
#include <string>

#include <cubutterfly/cubutterfly_b200.h>

#include "block_ops.hpp"
#include "gated_delta.hpp"
#include "qk_norm.hpp"

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

// ---- gated delta rule ---------------------------------------------------------------------------
template <typename Args>
void check_delta_heads(const Args* a) {
    require(a->k_heads >= 1 && a->heads >= 1 && a->k_dim >= 1 && a->v_dim >= 1,
            "gated delta: heads and their sizes must be at least 1");
    supported(a->heads <= 65536 && a->k_heads <= a->heads, "gated delta: at most 65536 heads, no more key heads than heads");
    require(a->heads % a->k_heads == 0, "gated delta: heads must be a multiple of k_heads");
    supported(a->k_dim <= cubf::kDeltaMaxDim && a->v_dim <= cubf::kDeltaMaxDim,
              "gated delta: k_dim and v_dim are limited to 128");
    require(std::isfinite(a->scale), "gated delta: scale must be finite");
}

cubf::HeadTensor head_tensor(const cubutterflyB200HeadTensor_t& t, size_t size, const char* what) {
    require(t.data != nullptr, what);
    require(element_aligned(t.data, size), what);
    return {t.data, t.batch, t.token, t.head};
}

template <typename Args, typename Call>
void delta_heads(const Args* a, Call& s) {
    check_delta_heads(a);
    s.k_heads = static_cast<int>(a->k_heads);
    s.heads = static_cast<int>(a->heads);
    s.k_dim = static_cast<int>(a->k_dim);
    s.v_dim = static_cast<int>(a->v_dim);
    s.scale = static_cast<float>(a->scale);
}

// ---- tensors apart from one another -----------------------------------------
struct Bytes {                   // an output, or another contiguous tensor
    uintptr_t from = 0, to = 0;
    Bytes(const void* p, size_t size) : from(reinterpret_cast<uintptr_t>(p)), to(p ? from + size : from) {}
};
bool meet(const Bytes& a, const Bytes& b) { return a.from < b.to && b.from < a.to; }

struct HeadSizes {
    size_t batch, tokens, heads, channels, size;
    size_t bytes() const { return batch * tokens * heads * channels * size; }
};
// `out` meets a batch row of `t`, from the row's first value to its last.
bool meet(const Bytes& out, const cubf::HeadTensor& t, const HeadSizes& n) {
    if (!t.p || n.bytes() == 0 || out.from == out.to) return false;
    const uintptr_t base = reinterpret_cast<uintptr_t>(t.p);
    const size_t row = ((n.tokens - 1) * t.token + (n.heads - 1) * t.head + n.channels) * n.size, step = t.batch * n.size;
    size_t b = 0;                // the first row that ends behind out's beginning
    if (base + row <= out.from) {
        if (step == 0) return false;
        b = (out.from - base - row) / step + 1;
    }
    return b < n.batch && base + b * step < out.to;
}
// `p`, contiguous, is `t` itself: read and written at the same places.
bool in_place(const void* p, const cubf::HeadTensor& t, const HeadSizes& n) {
    return p == t.p && (n.heads == 1 || t.head == n.channels) && (n.tokens == 1 || t.token == n.heads * n.channels) &&
           (n.batch == 1 || t.batch == n.tokens * n.heads * n.channels);
}

template <typename Args, typename Call>
void delta_gates(const Args* a, BlockType block, Call& s) {
    s.log_decay32 = vector_is_32(a->log_decay.data, a->log_decay_type, block, "gated delta log_decay_type");
    s.beta32 = vector_is_32(a->beta.data, a->beta_type, block, "gated delta beta_type");
    const size_t es = element(block);
    s.q = head_tensor(a->q, es, "gated delta: null or misaligned q");
    s.k = head_tensor(a->k, es, "gated delta: null or misaligned k");
    s.v = head_tensor(a->v, es, "gated delta: null or misaligned v");
    s.log_decay = head_tensor(a->log_decay, 2, "gated delta: null or misaligned log_decay");
    s.beta = head_tensor(a->beta, 2, "gated delta: null or misaligned beta");
}

// Without `tensors`: of what the workspace's size depends on.
cubf::GatedDeltaArgs delta_args(const cubutterflyB200GatedDelta_t* a, BlockType* block, bool tensors = true) {
    require(a != nullptr, "gated delta: null arguments");
    require(a->struct_size == sizeof(*a), "gated delta: struct_size does not match this library's");
    cubf::GatedDeltaArgs s{};
    delta_heads(a, s);
    supported(a->length <= cubf::kDeltaMaxLength, "gated delta: length is limited to 2^30 tokens");
    supported(a->batch <= (1u << 24) && a->sequences <= (1u << 30), "gated delta: too many sequences");
    require(!a->offsets || (a->batch == 1 && a->sequences >= 1),
            "gated delta: a packed batch has batch = 1 and at least one sequence");
    require(a->offsets || a->sequences == 0, "gated delta: sequences without offsets");
    *block = type_of(a->data_type, "gated delta data_type");
    s.batch = static_cast<int>(a->batch);
    s.length = static_cast<int>(a->length);
    s.sequences = static_cast<int>(a->sequences);
    s.initial = a->initial_state;
    s.offsets = a->offsets;
    constexpr int most = cubf::kDeltaWaitLimit;
    s.wait_limit = a->wait_limit == 0 ? most : std::clamp(a->wait_limit, 0, most);
    if (tensors && a->batch > 0 && a->length > 0) delta_gates(a, *block, s);
    // a CTA for each chunk of 64 tokens of each head
    const size_t chunks = a->offsets ? a->length / cubf::kDeltaChunk + a->sequences
                                     : a->batch * ((a->length + cubf::kDeltaChunk - 1) / cubf::kDeltaChunk);
    supported(chunks <= 0x7fffffffULL / a->heads, "gated delta: too many chunks and heads");
    const size_t states = a->offsets ? a->sequences : a->batch;
    supported(states <= 0x7fffffffULL / 16 / a->heads, "gated delta: too many sequences and heads");
    for (const void* p : {static_cast<const void*>(a->initial_state), static_cast<const void*>(a->offsets),
                          static_cast<const void*>(a->final_state), static_cast<const void*>(a->d_final_state),
                          static_cast<const void*>(a->d_initial_state)})
        require(element_aligned(p, 4), "gated delta: misaligned state or offsets");
    return s;
}

void delta_workspace(const cubutterflyB200GatedDelta_t* a, BlockType block, bool backward, cubf::GatedDeltaArgs& s) {
    require(a->workspace && a->workspace_bytes >= cubf::gated_delta_workspace(block, s, backward) &&
                element_aligned(a->workspace, 256),
            "gated delta: a 256-byte aligned workspace of the queried size is needed");
    s.workspace = a->workspace;
}

struct DeltaSizes {
    HeadSizes keys, values, decay, beta;
    size_t state, offsets;       // bytes
};
DeltaSizes delta_sizes(const cubf::GatedDeltaArgs& a, BlockType block) {
    const size_t batch = a.batch, length = a.length, heads = a.heads, states = a.offsets ? a.sequences : a.batch;
    const size_t k_heads = a.k_heads, k = a.k_dim, v = a.v_dim, es = element(block);
    return {{batch, length, k_heads, k, es},
            {batch, length, heads, v, es},
            {batch, length, heads, 1, a.log_decay32 ? 4 : es},
            {batch, length, heads, 1, a.beta32 ? 4 : es},
            states * heads * k * v * sizeof(float),
            a.offsets ? (a.sequences + size_t{1}) * sizeof(int) : 0};
}
// An output meets what both directions read.
bool delta_meets(const Bytes& out, const cubf::GatedDeltaArgs& a, const DeltaSizes& n) {
    return meet(out, a.q, n.keys) || meet(out, a.k, n.keys) || meet(out, a.v, n.values) || meet(out, a.log_decay, n.decay) ||
           meet(out, a.beta, n.beta) || meet(out, {a.initial, n.state}) || meet(out, {a.offsets, n.offsets});
}

// ---- norm of queries and keys -------------------------------------------------------------------
// What the workspace's size depends on.
cubf::QkNormArgs qk_sizes(const cubutterflyB200QkNorm_t* a) {
    require(a != nullptr, "qk norm: null arguments");
    require(a->struct_size == sizeof(*a), "qk norm: struct_size does not match this library's");
    require(a->dim >= 1, "qk norm: heads and their size must be at least 1");
    supported(a->dim <= cubf::kQkNormMaxDim, "qk norm: dim is limited to 256");
    supported(a->batch == 0 || a->tokens <= (size_t{1} << 40) / a->batch, "qk norm: too many tokens");
    cubf::QkNormArgs n{};
    n.batch = a->batch;
    n.tokens = a->tokens;
    n.dim = static_cast<int>(a->dim);
    n.q_weight = a->q_weight;
    n.k_weight = a->k_weight;
    n.parts = cubf::qk_norm_parts(n);
    return n;
}
cubf::QkNormArgs qk_args(const cubutterflyB200QkNorm_t* a, BlockType* block) {
    cubf::QkNormArgs n = qk_sizes(a);
    require(a->q_heads >= 1 && a->k_heads >= 1, "qk norm: heads and their size must be at least 1");
    supported(a->q_heads <= 65536 && a->k_heads <= 65536, "qk norm: at most 65536 heads");
    require(std::isfinite(a->epsilon) && a->epsilon >= 0, "qk norm: epsilon must be finite and not negative");
    require((a->flags & ~7) == 0, "qk norm: unknown flags");
    require(a->rotary % 2 == 0 && a->rotary <= a->dim, "qk norm: rotary must be even and at most dim");
    require((a->rotary > 0) == (a->positions != nullptr) && (a->rotary > 0) == (a->frequencies != nullptr),
            "qk norm: rotary, positions and frequencies go together");
    require(a->rotary == 0 || (a->positions_period >= 1 && a->axis_count >= 1 && a->axis_count <= 0x7fffffffULL),
            "qk norm: positions need a period and an axis");
    require(a->axes || a->axis_count <= 1, "qk norm: several axes of positions need axes");
    *block = type_of(a->data_type, "qk norm data_type");
    n.q_heads = static_cast<int>(a->q_heads);
    n.k_heads = static_cast<int>(a->k_heads);
    n.rotary = static_cast<int>(a->rotary);
    n.axis_count = static_cast<int>(a->axis_count);
    n.positions_axis = a->positions_axis;
    n.positions_period = a->positions_period;
    n.eps = static_cast<float>(a->epsilon);
    n.length = a->flags & CUBUTTERFLY_B200_QK_LENGTH;
    n.interleaved = a->flags & CUBUTTERFLY_B200_QK_INTERLEAVED;
    n.positions64 = a->flags & CUBUTTERFLY_B200_QK_POSITIONS64;
    require(element_aligned(a->positions, n.positions64 ? 8 : 4) && element_aligned(a->frequencies, 4) &&
                element_aligned(a->axes, 4),
            "qk norm: misaligned positions, frequencies or axes");
    n.positions = a->positions;
    n.frequencies = a->frequencies;
    n.axes = a->axes;
    n.q_weight32 = vector_is_32(a->q_weight, a->q_weight_type, *block, "qk norm q_weight_type");
    n.k_weight32 = vector_is_32(a->k_weight, a->k_weight_type, *block, "qk norm k_weight_type");
    if (a->batch == 0 || a->tokens == 0) return n;
    n.q = head_tensor(a->q, element(*block), "qk norm: null or misaligned q");
    n.k = head_tensor(a->k, element(*block), "qk norm: null or misaligned k");
    return n;
}

size_t qk_workspace(const cubf::QkNormArgs& a) {
    if (!a.q_weight && !a.k_weight) return 0;
    return (static_cast<size_t>(a.parts) * 2 * a.dim * sizeof(float) + 15) / 16 * 16;
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

extern "C" cubutterflyStatus_t cubutterflyB200GatedDeltaGetWorkspaceSize(const cubutterflyB200GatedDelta_t* args,
                                                                        int backward, size_t* bytes) {
    return guarded([&] {
        BlockType block;
        const cubf::GatedDeltaArgs a = delta_args(args, &block, false);
        require(bytes != nullptr, "gated delta: null size");
        *bytes = a.batch == 0 || a.length == 0 ? 0 : cubf::gated_delta_workspace(block, a, backward != 0);
    });
}

extern "C" cubutterflyStatus_t cubutterflyB200GatedDeltaForward(const cubutterflyB200GatedDelta_t* args,
                                                               cudaStream_t stream) {
    return guarded([&] {
        BlockType block;
        cubf::GatedDeltaArgs a = delta_args(args, &block);
        supported(a.length > 0 || a.batch == 0, "gated delta: of zero tokens the final states are the initial ones");
        if (a.batch == 0) return;
        require(args->o && element_aligned(args->o, element(block)), "gated delta: null or misaligned o");
        require(args->final_state != nullptr, "gated delta: null final_state");
        a.o = args->o;
        a.last = args->final_state;
        delta_workspace(args, block, false, a);
        const DeltaSizes n = delta_sizes(a, block);
        const Bytes o(a.o, n.values.bytes()), last(a.last, n.state);
        require(!delta_meets(o, a, n) && !delta_meets(last, a, n) && !meet(o, last),
                "gated delta: o and final_state must not alias an input or one another");
        check(cubf::launch_gated_delta(block, a, false, stream), "gated delta launch");
    });
}

extern "C" cubutterflyStatus_t cubutterflyB200GatedDeltaBackward(const cubutterflyB200GatedDelta_t* args,
                                                                cudaStream_t stream) {
    return guarded([&] {
        BlockType block;
        cubf::GatedDeltaArgs a = delta_args(args, &block);
        supported(a.length > 0 && a.batch > 0, "gated delta: the backward of zero tokens is the caller's zeros");
        const size_t es = element(block);
        a.d_o = head_tensor(args->d_o, es, "gated delta: null or misaligned d_o");
        require(args->d_q && args->d_k && args->d_v && args->d_log_decay && args->d_beta, "gated delta: null gradient");
        for (const void* p : {static_cast<const void*>(args->d_q), static_cast<const void*>(args->d_k),
                              static_cast<const void*>(args->d_v)})
            require(element_aligned(p, es), "gated delta: misaligned gradient");
        require(element_aligned(args->d_log_decay, a.log_decay32 ? 4 : es) && element_aligned(args->d_beta, a.beta32 ? 4 : es),
                "gated delta: misaligned gradient of a gate");
        a.d_last = args->d_final_state;
        a.d_q = args->d_q;
        a.d_k = args->d_k;
        a.d_v = args->d_v;
        a.d_log_decay = args->d_log_decay;
        a.d_beta = args->d_beta;
        a.d_initial = args->d_initial_state;
        delta_workspace(args, block, true, a);
        const DeltaSizes n = delta_sizes(a, block);
        const Bytes outs[] = {{a.d_q, n.keys.bytes()},          {a.d_k, n.keys.bytes()}, {a.d_v, n.values.bytes()},
                              {a.d_log_decay, n.decay.bytes()}, {a.d_beta, n.beta.bytes()}, {a.d_initial, n.state}};
        for (const Bytes& out : outs) {
            require(!delta_meets(out, a, n) && !meet(out, a.d_o, n.values) && !meet(out, {a.d_last, n.state}),
                    "gated delta: a gradient must not alias a tensor that is read");
            for (const Bytes& other : outs)
                require(&out == &other || !meet(out, other), "gated delta: gradients must not alias one another");
        }
        check(cubf::launch_gated_delta(block, a, true, stream), "gated delta backward launch");
    });
}

extern "C" cubutterflyStatus_t cubutterflyB200GatedDeltaStep(const cubutterflyB200GatedDeltaStep_t* a,
                                                            cudaStream_t stream) {
    return guarded([&] {
        require(a != nullptr, "gated delta step: null arguments");
        require(a->struct_size == sizeof(*a), "gated delta step: struct_size does not match this library's");
        cubf::GatedDeltaStepArgs s{};
        delta_heads(a, s);
        supported(a->batch <= 0x7fffffffULL && a->pool <= 0x7fffffffULL, "gated delta step: too many requests or slots");
        const BlockType block = type_of(a->data_type, "gated delta step data_type");
        if (a->batch == 0) return;
        delta_gates(a, block, s);
        require(a->o && element_aligned(a->o, element(block)), "gated delta step: null or misaligned o");
        require((a->state && a->new_state) || a->pool == 0, "gated delta step: null state");
        require(a->slots || a->pool >= a->batch, "gated delta step: without slots the pool needs a state per request");
        for (const void* p : {static_cast<const void*>(a->state), static_cast<const void*>(a->new_state),
                              static_cast<const void*>(a->slots)})
            require(element_aligned(p, 4), "gated delta step: misaligned state or slots");
        // in place, or apart, as in the gated scan's step
        const uintptr_t from = reinterpret_cast<uintptr_t>(a->state), to = reinterpret_cast<uintptr_t>(a->new_state);
        const size_t bytes = a->pool * a->heads * a->k_dim * a->v_dim * sizeof(float);
        require(from == to || from + bytes <= to || to + bytes <= from,
                "gated delta step: new_state must be state or not overlap it");
        s.state = a->state;
        s.new_state = a->new_state;
        s.slots = a->slots;
        s.o = a->o;
        s.batch = a->batch;
        s.pool = a->pool;
        const size_t es = element(block), heads = a->heads;
        const HeadSizes keys{a->batch, 1, a->k_heads, a->k_dim, es}, values{a->batch, 1, heads, a->v_dim, es};
        const Bytes o(s.o, values.bytes());
        require(!meet(o, s.q, keys) && !meet(o, s.k, keys) && (in_place(s.o, s.v, values) || !meet(o, s.v, values)) &&
                    !meet(o, s.log_decay, {a->batch, 1, heads, 1, s.log_decay32 ? 4 : es}) &&
                    !meet(o, s.beta, {a->batch, 1, heads, 1, s.beta32 ? 4 : es}) && !meet(o, {s.state, bytes}) &&
                    !meet(o, {s.new_state, bytes}),
                "gated delta step: o must not alias another tensor (v itself excepted)");
        check(cubf::launch_gated_delta_step(block, s, stream), "gated delta step launch");
    });
}

extern "C" cubutterflyStatus_t cubutterflyB200QkNormForward(const cubutterflyB200QkNorm_t* args, cudaStream_t stream) {
    return guarded([&] {
        BlockType block;
        cubf::QkNormArgs a = qk_args(args, &block);
        if (a.batch == 0 || a.tokens == 0) return;
        const size_t es = element(block);
        require(args->q_out && args->k_out && element_aligned(args->q_out, es) && element_aligned(args->k_out, es),
                "qk norm: null or misaligned output");
        a.q_out = args->q_out;
        a.k_out = args->k_out;
        const HeadSizes q{a.batch, a.tokens, args->q_heads, args->dim, es}, k{a.batch, a.tokens, args->k_heads, args->dim, es};
        const Bytes qs(a.q_out, q.bytes()), ks(a.k_out, k.bytes());
        require(!meet(qs, a.q, q) && !meet(qs, a.k, k) && !meet(ks, a.q, q) && !meet(ks, a.k, k) && !meet(qs, ks),
                "qk norm: an output must not alias another tensor");
        check(cubf::launch_qk_norm(block, a, false, stream), "qk norm launch");
    });
}

extern "C" cubutterflyStatus_t cubutterflyB200QkNormGetWorkspaceSize(const cubutterflyB200QkNorm_t* args, size_t* bytes) {
    return guarded([&] {
        const cubf::QkNormArgs a = qk_sizes(args);
        require(bytes != nullptr, "qk norm: null size");
        *bytes = qk_workspace(a);
    });
}

extern "C" cubutterflyStatus_t cubutterflyB200QkNormBackward(const cubutterflyB200QkNorm_t* args, cudaStream_t stream) {
    return guarded([&] {
        BlockType block;
        cubf::QkNormArgs a = qk_args(args, &block);
        supported(a.batch > 0 && a.tokens > 0, "qk norm: the backward of zero tokens is the caller's zeros");
        const size_t es = element(block);
        a.d_q_out = head_tensor(args->d_q_out, es, "qk norm: null or misaligned d_q_out");
        a.d_k_out = head_tensor(args->d_k_out, es, "qk norm: null or misaligned d_k_out");
        require(args->d_q && args->d_k && element_aligned(args->d_q, es) && element_aligned(args->d_k, es),
                "qk norm: null or misaligned gradient");
        require((args->d_q_weight != nullptr) == (args->q_weight != nullptr) &&
                    (args->d_k_weight != nullptr) == (args->k_weight != nullptr),
                "qk norm: every weight needs its gradient");
        require(element_aligned(args->d_q_weight, a.q_weight32 ? 4 : es) && element_aligned(args->d_k_weight, a.k_weight32 ? 4 : es),
                "qk norm: misaligned gradient of a weight");
        require(qk_workspace(a) == 0 || (args->workspace && args->workspace_bytes >= qk_workspace(a) &&
                                         element_aligned(args->workspace, 16)),
                "qk norm: the backward needs a 16-byte aligned workspace of the queried size");
        a.d_q = args->d_q;
        a.d_k = args->d_k;
        a.d_q_weight = args->d_q_weight;
        a.d_k_weight = args->d_k_weight;
        a.partials = static_cast<float*>(args->workspace);
        // a head's gradient may take its own place, or that of the gradient it comes from
        const HeadSizes q{a.batch, a.tokens, args->q_heads, args->dim, es}, k{a.batch, a.tokens, args->k_heads, args->dim, es};
        const Bytes qs(a.d_q, q.bytes()), ks(a.d_k, k.bytes());
        auto apart = [](const void* p, const Bytes& out, const cubf::HeadTensor& t, const HeadSizes& n) {
            return in_place(p, t, n) || !meet(out, t, n);
        };
        require(apart(a.d_q, qs, a.q, q) && apart(a.d_q, qs, a.d_q_out, q) && apart(a.d_k, ks, a.k, k) &&
                    apart(a.d_k, ks, a.d_k_out, k) && !meet(qs, a.k, k) && !meet(qs, a.d_k_out, k) && !meet(ks, a.q, q) &&
                    !meet(ks, a.d_q_out, q) && !meet(qs, ks),
                "qk norm: a gradient must not alias another tensor (that of its own head excepted)");
        check(cubf::launch_qk_norm(block, a, true, stream), "qk norm backward launch");
    });
}
