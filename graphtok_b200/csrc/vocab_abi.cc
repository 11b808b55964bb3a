// extern "C" entries of the operators between token ids and a model's vocabulary-wide tables; see include/gtok.h for the contract.
#include "../../include/gtok.h"

#include <cuda_runtime.h>

#include <cmath>

#include "vocab_next.h"
#include "vocab_ops.h"

namespace gtok {
void set_last_error(const char* message);
}

namespace {

constexpr int64_t kMostRows = (1ll << 31) - 1024;

int32_t refuse(const char* why) {
    gtok::set_last_error(why);
    return -1;
}
int32_t done(const char* error) { return error ? refuse(error) : 0; }

int element(int type) { return type == gtok::kF32 ? 4 : 2; }

// The current device; -1 with a message where it is no B200.
int device() {
    int d = 0, major = 0;
    if (cudaGetDevice(&d) != cudaSuccess || cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, d) != cudaSuccess) {
        cudaGetLastError();
        return refuse("no GPU");
    }
    if (major != 10) return refuse("the current device is no B200");
    // A thread that has called nothing yet, such as one of torch's for backward passes, has no context for the driver's calls until this.
    static thread_local int ready = -1;
    if (ready != d) {
        if (cudaSetDevice(d) != cudaSuccess) {
            cudaGetLastError();
            return refuse("the current device cannot be used");
        }
        ready = d;
    }
    return d;
}

// An address that the current device's kernels may use: its own memory, or memory that it shares with the host.
bool usable(const void* at, int d) {
    cudaPointerAttributes a;
    if (cudaPointerGetAttributes(&a, at) != cudaSuccess) {
        cudaGetLastError();
        return false;
    }
    return (a.type == cudaMemoryTypeDevice && a.device == d) || a.type == cudaMemoryTypeManaged;
}

bool floats(const void* at, int d) { return at && reinterpret_cast<uintptr_t>(at) % 4 == 0 && usable(at, d); }

const char* check(const gtok_x_matrix* m, int d) {
    if (!m) return "a matrix is missing";
    if (m->type != gtok::kF32 && m->type != gtok::kBF16 && m->type != gtok::kF16) return "a matrix's type is none of fp32, bf16, fp16";
    if (m->rows < 0 || m->rows > kMostRows || m->cols < 1 || m->cols > (1 << 20)) return "a matrix's rows or columns are out of range";
    if (m->stride < 0 || m->stride > (1ll << 35)) return "a matrix's row stride is out of range";
    if (m->rows && !m->data) return "a matrix has no data";
    if (reinterpret_cast<uintptr_t>(m->data) % element(m->type)) return "a matrix's data is not aligned to its elements";
    if (m->rows && !usable(m->data, d)) return "a matrix's data is not in the current device's memory";
    return nullptr;
}
// Where rows are written they must not lie over one another.
const char* check_out(const gtok_x_matrix* m, int d) {
    if (const char* e = check(m, d)) return e;
    return m->rows > 1 && m->stride < m->cols ? "rows of an output lie over one another" : nullptr;
}
const char* check_ids(const void* ids, int32_t bits, int64_t n, int d) {
    if (bits != 32 && bits != 64) return "ids have 32 or 64 bits";
    if (n < 0 || n > kMostRows) return "the number of ids is out of range";
    if (n && (!ids || reinterpret_cast<uintptr_t>(ids) % (bits / 8) || !usable(ids, d))) return "ids are missing, not aligned, or not in the current device's memory";
    return nullptr;
}
const char* check_workspace(const void* at, uint64_t bytes, uint64_t need, int d) {
    if (!need) return nullptr;
    if (bytes < need) return "the workspace is too small";
    if (!at || reinterpret_cast<uintptr_t>(at) % 256 || !usable(at, d)) return "the workspace is missing, not aligned to 256 bytes, or not in the current device's memory";
    return nullptr;
}

gtok::Matrix matrix(const gtok_x_matrix& m) {
    gtok::Matrix r;
    r.data = m.data;
    r.rows = m.rows;
    r.cols = m.cols;
    r.stride = m.stride;
    r.type = m.type;
    return r;
}
gtok::Ids make_ids(const void* data, int32_t bits, int64_t stride) {
    gtok::Ids r;
    r.data = data;
    r.bits = bits;
    r.stride = stride;
    return r;
}

// Sizes and numbers of a loss; what needs no address.
const char* check_sizes(const gtok_x_vocab_loss* a) {
    const gtok_x_matrix &h = a->hidden, &w = a->weight;
    if ((h.type != gtok::kBF16 && h.type != gtok::kF16) || h.type != w.type) return "hidden states and table are both bf16 or both fp16";
    if (h.cols != w.cols) return "hidden states and table have different widths";
    if (h.cols < 1 || h.cols > (1 << 16)) return "the width is out of range";
    // (a tile of the table's gradient sums over all rows, and is waited for in the kernel: 2^28 of them take a second)
    if (h.rows < 0 || h.rows > (1ll << 28) || w.rows < 1 || w.rows > (1ll << 30)) return "rows or vocabulary are out of range";
    if ((h.rows / 256 + 1) * (w.rows / 256 + 1) > (1 << 28)) return "rows times vocabulary are out of range";
    if (a->entries < 0 || a->entries > gtok::kMaxEntries) return "a teacher's row has 1 to 1024 entries";
    // (log2(e) / T is a number of fp32 for every normal one)
    if (!(a->temperature > 0.f) || !std::isnormal(a->temperature)) return "the temperature must be positive, finite and at least 2^-126";
    return nullptr;
}

gtok::LossCall loss_call(const gtok_x_vocab_loss* a) {
    gtok::LossCall c;
    c.hidden = matrix(a->hidden);
    c.weight = matrix(a->weight);
    c.targets = make_ids(a->targets, a->target_bits, a->target_stride);
    c.entries = a->entries;
    c.teacher = matrix(a->teacher_logits);
    c.ignore = a->ignore;
    c.temperature = a->temperature;
    c.losses = a->losses;
    c.lse = a->lse;
    c.total = a->total;
    c.mean = a->mean != 0;
    c.grad = a->grad;
    c.grad_stride = a->mean ? 0 : a->grad_stride;
    c.kept = a->kept;
    c.d_hidden = matrix(a->d_hidden);
    c.d_weight = matrix(a->d_weight);
    c.workspace = a->workspace;
    c.workspace_bytes = a->workspace_bytes;
    c.stream = static_cast<cudaStream_t>(a->cuda_stream);
    return c;
}

// `values`: hidden states and targets are read, not only what a forward pass kept of them.
const char* check_loss(const gtok_x_vocab_loss* a, int d, bool values) {
    if (const char* e = check_sizes(a)) return e;
    if (const char* e = check(&a->weight, d)) return e;
    if (a->weight.rows > 1 && a->weight.stride < a->weight.cols) return "rows of the table lie over one another";
    if (values) {
        if (const char* e = check(&a->hidden, d)) return e;
        if (const char* e = check_ids(a->targets, a->target_bits, a->hidden.rows, d)) return e;
        if (a->entries) {
            if (const char* e = check(&a->teacher_logits, d)) return e;
            if (a->teacher_logits.rows != a->hidden.rows || a->teacher_logits.cols != a->entries) return "the teacher's logits have another shape than its ids";
            if (a->target_stride < 0) return "the stride of the teacher's ids is out of range";
        }
    }
    if (a->kept && a->hidden.rows) {
        if (reinterpret_cast<uintptr_t>(a->kept) % 256 || !usable(a->kept, d)) return "`kept` is not aligned to 256 bytes or not in the current device's memory";
        if (a->kept_bytes < gtok::loss_kept(loss_call(a))) return "`kept` is too small";
    }
    return nullptr;
}

const char* check_gradient(const gtok_x_matrix* m, const gtok_x_matrix& of, int d) {
    if (!m->data) return nullptr;
    if (m->type != of.type || m->rows != of.rows || m->cols != of.cols) return "a gradient has another shape or type than what it is of";
    return check_out(m, d);
}

const char* check_table4_sizes(int64_t vocab, int64_t width, int64_t group) {
    if (vocab < 1 || vocab > (1 << 24) || width < 1 || width > (1 << 16)) return "a table's rows or columns are out of range";
    if (group != 32 && (group < 64 || group > (1 << 16) || group % 64)) return "a group has 32 columns or a multiple of 64";
    return nullptr;
}
const char* check_table4(const gtok_x_table4* t, int d) {
    if (!t) return "a table is missing";
    if (t->type != gtok::kBF16 && t->type != gtok::kF16) return "a table's scales are bf16 or fp16";
    if (const char* e = check_table4_sizes(t->vocab, t->width, t->group)) return e;
    if (t->zeros != 0 && t->zeros != 1) return "zeros is 0 or 1";
    if (t->bytes < gtok::table4_plan(t->vocab, t->width, t->group, t->zeros != 0).bytes) return "the table's memory is too small";
    if (!t->data || reinterpret_cast<uintptr_t>(t->data) % 256 || !usable(t->data, d)) return "the table's memory is missing, not aligned to 256 bytes, or not in the current device's memory";
    return nullptr;
}
gtok::Table4 table4(const gtok_x_table4& t) {
    gtok::Table4 r;
    r.data = t.data;
    r.vocab = t.vocab;
    r.width = t.width;
    r.group = t.group;
    r.type = t.type;
    r.zeros = t.zeros != 0;
    return r;
}

// Logits: rows as wide as a vocabulary.
const char* check_logits(const gtok_x_matrix* m, int d) {
    if (m->cols < 1 || m->cols > (1 << 24)) return "a vocabulary has 1 to 2^24 ids";
    if (m->rows > (1 << 20)) return "the number of rows is out of range";
    gtok_x_matrix shape = *m;
    shape.cols = 1;                            // (a matrix of fewer columns than a vocabulary may have ids is meant elsewhere)
    return check(&shape, d);
}
// An optional list of numbers of 4 bytes.
bool words(const void* at, int d) { return !at || floats(at, d); }

}  // namespace

extern "C" {

int64_t gtok_x_table4_bytes(int64_t vocab, int64_t width, int64_t group, int32_t zeros) {
    if (const char* e = check_table4_sizes(vocab, width, group)) return refuse(e);
    return static_cast<int64_t>(gtok::table4_plan(vocab, width, group, zeros != 0).bytes);
}

int32_t gtok_x_table4_pack(const gtok_x_table4* table, const uint8_t* codes, int64_t codes_stride, const gtok_x_matrix* scales, const uint8_t* zeros, int64_t zeros_stride,
                           void* cuda_stream) {
    try {
        const int d = device();
        if (d < 0) return -1;
        if (const char* e = check_table4(table, d)) return refuse(e);
        if (!codes || !usable(codes, d)) return refuse("the codes are missing or not in the current device's memory");
        if (codes_stride < 0 || codes_stride > (1ll << 35) || zeros_stride < 0 || zeros_stride > (1ll << 35)) return refuse("the stride of the codes or zeros is out of range");
        if (const char* e = check(scales, d)) return refuse(e);
        if (scales->type != table->type || scales->rows != table->vocab || scales->cols != (table->width + table->group - 1) / table->group)
            return refuse("the scales have another shape or type than the table's");
        if (table->zeros && (!zeros || !usable(zeros, d))) return refuse("the zeros are missing or not in the current device's memory");
        return done(gtok::pack_table(table4(*table), codes, codes_stride, matrix(*scales), zeros, zeros_stride, static_cast<cudaStream_t>(cuda_stream)));
    } catch (...) { return refuse("an internal error"); }
}

int32_t gtok_x_table4_quantize(const gtok_x_table4* table, const gtok_x_matrix* weight, void* cuda_stream) {
    try {
        const int d = device();
        if (d < 0) return -1;
        if (const char* e = check_table4(table, d)) return refuse(e);
        if (const char* e = check(weight, d)) return refuse(e);
        if (weight->rows != table->vocab || weight->cols != table->width) return refuse("the weights have another shape than the table");
        return done(gtok::quantize_table(table4(*table), matrix(*weight), static_cast<cudaStream_t>(cuda_stream)));
    } catch (...) { return refuse("an internal error"); }
}

int32_t gtok_x_table4_logits(const gtok_x_matrix* hidden, const gtok_x_table4* table, const gtok_x_matrix* out, void* cuda_stream) {
    try {
        const int d = device();
        if (d < 0) return -1;
        if (const char* e = check_table4(table, d)) return refuse(e);
        if (const char* e = check(hidden, d)) return refuse(e);
        if (hidden->cols != table->width || hidden->type != table->type) return refuse("the hidden states have another width or type than the table");
        if (!out || out->cols != table->vocab || out->rows != hidden->rows) return refuse("the logits have another shape than hidden states and table");
        if (out->type != gtok::kF32 && out->type != table->type) return refuse("logits are fp32 or of the table's type");
        if (const char* e = check_logits(out, d)) return refuse(e);
        if (out->rows > 1 && out->stride < out->cols) return refuse("rows of an output lie over one another");
        return done(gtok::table_logits(matrix(*hidden), table4(*table), matrix(*out), static_cast<cudaStream_t>(cuda_stream)));
    } catch (...) { return refuse("an internal error"); }
}

int32_t gtok_x_adjust_logits(const gtok_x_adjustment* a) {
    try {
        const int d = device();
        if (d < 0) return -1;
        if (!a) return refuse("arguments are missing");
        const int64_t n = a->logits.rows, vocab = a->logits.cols;
        if (const char* e = check_logits(&a->logits, d)) return refuse(e);
        if (const char* e = check_logits(&a->out, d)) return refuse(e);
        if (a->out.rows != n || a->out.cols != vocab || a->out.type != a->logits.type) return refuse("the output has another shape or type than the logits");
        if (n > 1 && a->out.stride < vocab) return refuse("rows of an output lie over one another");
        if (n > 1 && a->out.data == a->logits.data && a->out.stride != a->logits.stride) return refuse("logits that are changed in place have one stride");
        if (a->offsets) {
            if (const char* e = check_ids(a->ids, a->id_bits, a->n_ids, d)) return refuse(e);
            if (const char* e = check_ids(a->offsets, 32, n + 1, d)) return refuse(e);
        }
        if (!words(a->prompt_lengths, d) || !words(a->repetition, d) || !words(a->presence, d) || !words(a->frequency, d))
            return refuse("prompt lengths or penalties are not aligned or not in the current device's memory");
        if (a->entries < 0 || a->entries > gtok::kMaxBiases) return refuse("a row has at most 1024 biases");
        if (a->bias_stride < 0 || a->bias_stride > (1ll << 35)) return refuse("the stride of the biases is out of range");
        if (n && a->entries && (!floats(a->bias_ids, d) || !floats(a->bias, d))) return refuse("biases are missing, not aligned, or not in the current device's memory");
        if (!words(a->allowed, d) || !words(a->allowed_rows, d)) return refuse("masks are not aligned or not in the current device's memory");
        if (a->allowed && (a->allowed_count < 0 || a->allowed_stride < 0 || a->allowed_stride > (1ll << 35))) return refuse("number or stride of the masks are out of range");
        gtok::AdjustCall c;
        c.logits = matrix(a->logits);
        c.out = matrix(a->out);
        c.ids = make_ids(a->ids, a->id_bits, 1);
        c.n_ids = a->n_ids;
        c.offsets = a->offsets;
        c.prompt_lengths = a->prompt_lengths;
        c.repetition = a->repetition;
        c.presence = a->presence;
        c.frequency = a->frequency;
        c.one_repetition = a->one_repetition;
        c.one_presence = a->one_presence;
        c.one_frequency = a->one_frequency;
        c.entries = a->entries;
        c.bias_ids = a->bias_ids;
        c.bias = a->bias;
        c.bias_stride = a->bias_stride;
        c.allowed = a->allowed;
        c.allowed_rows = a->allowed_rows;
        c.allowed_count = a->allowed_count;
        c.allowed_stride = a->allowed_stride;
        c.stream = static_cast<cudaStream_t>(a->cuda_stream);
        return done(gtok::adjust_logits(c));
    } catch (...) { return refuse("an internal error"); }
}

int32_t gtok_x_sample(const gtok_x_draw* a) {
    try {
        const int d = device();
        if (d < 0) return -1;
        if (!a) return refuse("arguments are missing");
        if (const char* e = check_logits(&a->logits, d)) return refuse(e);
        if (a->u_bits != 32 && a->u_bits != 64) return refuse("random numbers have 32 or 64 bits");
        if (a->logits.rows) {
            if (!a->u || reinterpret_cast<uintptr_t>(a->u) % (a->u_bits / 8) || !usable(a->u, d)) return refuse("random numbers are missing, not aligned, or not in the current device's memory");
            if (!floats(a->ids, d) || !floats(a->logprobs, d)) return refuse("ids or logprobs are missing, not aligned, or not in the current device's memory");
        }
        if (!words(a->temperature, d) || !words(a->top_k, d) || !words(a->top_p, d) || !words(a->min_p, d))
            return refuse("temperature, top_k, top_p or min_p are not aligned or not in the current device's memory");
        gtok::SampleCall c;
        c.logits = matrix(a->logits);
        c.u = a->u;
        c.wide_u = a->u_bits == 64;
        c.temperature = a->temperature;
        c.top_k = a->top_k;
        c.top_p = a->top_p;
        c.min_p = a->min_p;
        c.one_temperature = a->one_temperature;
        c.one_top_k = a->one_top_k;
        c.one_top_p = a->one_top_p;
        c.one_min_p = a->one_min_p;
        c.ids = a->ids;
        c.logprobs = a->logprobs;
        c.stream = static_cast<cudaStream_t>(a->cuda_stream);
        return done(gtok::sample(c));
    } catch (...) { return refuse("an internal error"); }
}

int32_t gtok_x_embed(const void* ids, int32_t id_bits, int64_t n, const gtok_x_matrix* table, float scale, const gtok_x_matrix* out, void* cuda_stream) {
    try {
        const int d = device();
        if (d < 0) return -1;
        if (const char* e = check_ids(ids, id_bits, n, d)) return refuse(e);
        if (const char* e = check(table, d)) return refuse(e);
        if (const char* e = check_out(out, d)) return refuse(e);
        if (out->rows != n || out->cols != table->cols || out->type != table->type) return refuse("the output has another shape or type than the looked up rows");
        return done(gtok::embed(make_ids(ids, id_bits, 1), n, matrix(*table), scale, matrix(*out), static_cast<cudaStream_t>(cuda_stream)));
    } catch (...) { return refuse("an internal error"); }
}

int64_t gtok_x_embed_grad_workspace(int64_t n, int64_t vocab, int64_t width) {
    if (n < 0 || n > kMostRows || vocab < 0 || vocab > kMostRows || width < 1 || width > (1 << 20)) return refuse("a size is out of range");
    return static_cast<int64_t>(gtok::embed_grad_workspace(n, vocab, width));
}

int32_t gtok_x_embed_grad(const void* ids, int32_t id_bits, int64_t n, const gtok_x_matrix* grad, float scale, const gtok_x_matrix* out, int32_t accumulate,
                          void* workspace, uint64_t workspace_bytes, void* cuda_stream) {
    try {
        const int d = device();
        if (d < 0) return -1;
        if (const char* e = check_ids(ids, id_bits, n, d)) return refuse(e);
        if (const char* e = check(grad, d)) return refuse(e);
        if (const char* e = check_out(out, d)) return refuse(e);
        if (grad->rows != n || grad->cols != out->cols || grad->type != out->type) return refuse("the gradient has another shape or type than the table's");
        if (const char* e = check_workspace(workspace, workspace_bytes, gtok::embed_grad_workspace(n, out->rows, out->cols), d)) return refuse(e);
        return done(gtok::embed_grad(make_ids(ids, id_bits, 1), n, matrix(*grad), scale, matrix(*out), accumulate != 0, workspace, workspace_bytes,
                                     static_cast<cudaStream_t>(cuda_stream)));
    } catch (...) { return refuse("an internal error"); }
}

int32_t gtok_x_next_targets(const int32_t* ids, int64_t n, const int32_t* doc_offsets, int64_t n_docs, const uint8_t* loss_mask, int32_t ignore, int32_t* out,
                            void* cuda_stream) {
    try {
        const int d = device();
        if (d < 0) return -1;
        if (const char* e = check_ids(ids, 32, n, d)) return refuse(e);
        if (const char* e = check_ids(out, 32, n, d)) return refuse(e);
        if (n_docs < 0) return refuse("the number of documents is out of range");
        if (const char* e = check_ids(doc_offsets, 32, n_docs + 1, d)) return refuse(e);
        if (n && loss_mask && !usable(loss_mask, d)) return refuse("the mask is not in the current device's memory");
        return done(gtok::next_targets(ids, n, doc_offsets, n_docs, loss_mask, ignore, out, static_cast<cudaStream_t>(cuda_stream)));
    } catch (...) { return refuse("an internal error"); }
}

int64_t gtok_x_vocab_loss_workspace(const gtok_x_vocab_loss* args, int32_t backward) {
    if (!args) return refuse("arguments are missing");
    if (const char* e = check_sizes(args)) return refuse(e);
    return static_cast<int64_t>(gtok::loss_workspace(loss_call(args), backward != 0));
}

int64_t gtok_x_vocab_loss_kept(const gtok_x_vocab_loss* args) {
    if (!args) return refuse("arguments are missing");
    if (const char* e = check_sizes(args)) return refuse(e);
    return static_cast<int64_t>(gtok::loss_kept(loss_call(args)));
}

int32_t gtok_x_vocab_loss_forward(const gtok_x_vocab_loss* args) {
    try {
        const int d = device();
        if (d < 0) return -1;
        if (!args) return refuse("arguments are missing");
        if (const char* e = check_loss(args, d, true)) return refuse(e);
        if (args->hidden.rows && (!floats(args->losses, d) || !floats(args->lse, d)))
            return refuse("losses or lse are missing, not aligned, or not in the current device's memory");
        if (args->total && !floats(args->total, d)) return refuse("the total is not aligned or not in the current device's memory");
        const gtok::LossCall c = loss_call(args);
        if (const char* e = check_workspace(args->workspace, args->workspace_bytes, gtok::loss_workspace(c, false), d)) return refuse(e);
        return done(gtok::loss_forward(c));
    } catch (...) { return refuse("an internal error"); }
}

int32_t gtok_x_vocab_loss_backward(const gtok_x_vocab_loss* args) {
    try {
        const int d = device();
        if (d < 0) return -1;
        if (!args) return refuse("arguments are missing");
        if (const char* e = check_loss(args, d, !args->kept)) return refuse(e);
        if (!args->d_hidden.data && !args->d_weight.data) return 0;
        if (args->hidden.rows && (!floats(args->lse, d) || !floats(args->grad, d)))
            return refuse("lse or the losses' gradient are missing, not aligned, or not in the current device's memory");
        if (args->grad_stride < 0) return refuse("the stride of the losses' gradient is out of range");
        if (const char* e = check_gradient(&args->d_hidden, args->hidden, d)) return refuse(e);
        if (const char* e = check_gradient(&args->d_weight, args->weight, d)) return refuse(e);
        const gtok::LossCall c = loss_call(args);
        if (const char* e = check_workspace(args->workspace, args->workspace_bytes, gtok::loss_workspace(c, true), d)) return refuse(e);
        return done(gtok::loss_backward(c));
    } catch (...) { return refuse("an internal error"); }
}

}  // extern "C"
