// The operators on logits behind the C ABI: argument checks, scratch and launches.
#include "pcu_checks.hpp"

namespace pcu {

static_assert(kLogitMaxVocab == PCU_LOGITS_MAX_VOCAB && kLogitMaxK == PCU_LOGITS_MAX_K, "one limit");
static_assert(kLogitF32 == PCU_F32 && kLogitF64 == PCU_F64 && kLogitBf16 == PCU_BF16 && kLogitF16 == PCU_F16,
              "one numbering");

static uint64_t logits_bytes(const pcu_logits &l)
{
    return strided_bytes(l.rows, l.vocab, l.stride, logit_size(l.dtype));
}

static pcu_status check_logits(Ctx *c, const char *what, const pcu_logits *l)
{
    constexpr uint64_t kMaxStride = (uint64_t)PCU_LOGITS_MAX_VOCAB << 8;
    if (!l || l->dtype > PCU_F16 || (l->rows && l->vocab && !l->data) ||
        !aligned(l->data, logit_size(l->dtype))) {
        c->fail("%s: invalid logits", what);
        return PCU_ERR_ARGUMENT;
    }
    if (l->vocab > PCU_LOGITS_MAX_VOCAB || l->rows > PCU_LOGITS_MAX_ROWS || l->stride > kMaxStride ||
        l->stride < l->vocab) {
        c->fail("%s: %llu rows of %llu logits, stride %llu: beyond the limits", what, (unsigned long long)l->rows,
                (unsigned long long)l->vocab, (unsigned long long)l->stride);
        return PCU_ERR_SHAPE;
    }
    return PCU_OK;
}

// Whether the kernels can work with a temperature: it and what they make of it have to be numbers in
// the statistics' type (the exponent's factor is log2(e) / T; a loss takes the square, in binary64).
static bool valid_temperature(uint32_t dtype, double temperature, bool squared)
{
    if (!(temperature > 0) || !std::isfinite(temperature))
        return false;
    if (dtype == PCU_F64)
        return std::isfinite(1.0 / temperature) &&
               (!squared || (temperature * temperature > 0 && std::isfinite(temperature * temperature)));
    const float t = (float)temperature;
    return t > 0 && std::isfinite(t) && std::isfinite(1.0f / t * (float)M_LOG2E);
}

pcu_status Ctx::op_top_logits(const pcu_logits *l, uint32_t k, double temperature, void *values,
                              int32_t *indices, void *log_sum)
{
    pcu_status st = check_logits(this, "top_logits", l);
    if (st)
        return st;
    if (k > PCU_LOGITS_MAX_K) {
        fail("top_logits: k %u is beyond %u", k, PCU_LOGITS_MAX_K);
        return PCU_ERR_SHAPE;
    }
    if ((l->rows && k && (!values || !indices)) || !valid_temperature(l->dtype, temperature, false)) {
        fail("top_logits: invalid argument");
        return PCU_ERR_ARGUMENT;
    }
    if (!aligned(values, logit_size(l->dtype)) || !aligned(indices, 4) || !aligned(log_sum, stat_size(l->dtype))) {
        fail("top_logits: an output is not aligned to its type");
        return PCU_ERR_ARGUMENT;
    }
    const Range in{l->data, logits_bytes(*l)};
    const Range v{values, l->rows * k * logit_size(l->dtype)}, i{indices, l->rows * k * 4},
        s{log_sum, l->rows * stat_size(l->dtype)};
    if (overlaps_any(v, {in, i, s}) || overlaps_any(i, {in, s}) || overlaps_any(s, {in})) {
        fail("top_logits: an output overlaps another tensor");
        return PCU_ERR_ARGUMENT;
    }
    unsigned long long *word;
    if ((st = add_node(NodeInfo{Prim::Native, l->rows, 0}, &word)))
        return st;
    if ((st = open_words()))
        return st;
    TopArgs g;
    g.logits = l->data;
    g.dtype = (int)l->dtype;
    g.rows = l->rows;
    g.stride = l->stride;
    g.vocab = (uint32_t)l->vocab;
    g.k = k;
    g.temperature = temperature;
    g.values = values;
    g.indices = indices;
    g.log_sum = log_sum;
    g.gate = gate_for(word);
    ProgramClose close;
    if (implicit_program && nodes.size() == 1)
        close_next = true; // a call of its own: its kernel ends the program
    if ((st = take_close(&close)))
        return st;
    bool closed = false;
    hipEvent_t t = timer_start(stream);
    st = hip(launch_top(stream, g, close, &closed), "top_logits launch");
    timer_stop(PCU_KERNEL_TOP_LOGITS, t, stream);
    if (!st && closed)
        closed_seq = ++pub_seq;
    return st;
}

pcu_status Ctx::op_distill(Distill mode, const pcu_logits *l, const pcu_distill *d, const void *log_sums_in,
                           const void *row_scale, void *loss, void *log_sums_out, void *grad,
                           uint64_t grad_cols, uint64_t grad_stride)
{
    pcu_status st = check_logits(this, "distill", l);
    if (st)
        return st;
    if (!d || d->teacher_dtype > PCU_F16 ||
        (l->rows && d->k && (!d->teacher_values || !d->teacher_indices)) ||
        !valid_temperature(l->dtype, d->temperature, mode != Distill::Backward) ||
        !valid_weight(l->dtype, d->distill_weight) || !valid_weight(l->dtype, d->label_weight) ||
        (l->rows && mode != Distill::Backward && !loss) || (l->rows && mode == Distill::Backward && !log_sums_in) ||
        (l->rows && grad_cols && mode != Distill::Loss && !grad)) {
        fail("distill: invalid argument");
        return PCU_ERR_ARGUMENT;
    }
    if (d->k > PCU_LOGITS_MAX_K) {
        fail("distill: %u entries a row are beyond %u", d->k, PCU_LOGITS_MAX_K);
        return PCU_ERR_SHAPE;
    }
    const uint64_t size = logit_size(l->dtype), stat = stat_size(l->dtype);
    if (mode != Distill::Loss &&
        (grad_cols < l->vocab || grad_stride < grad_cols || grad_stride > ((uint64_t)PCU_LOGITS_MAX_VOCAB << 8) ||
         grad_cols - l->vocab > PCU_LOGITS_MAX_VOCAB || !aligned(grad, size))) {
        fail("distill: a gradient of %llu columns, stride %llu, for %llu logits", (unsigned long long)grad_cols,
             (unsigned long long)grad_stride, (unsigned long long)l->vocab);
        return PCU_ERR_SHAPE;
    }
    if (!aligned(d->teacher_values, logit_size(d->teacher_dtype)) || !aligned(d->teacher_indices, 4) ||
        !aligned(d->teacher_log_sum, stat_size(d->teacher_dtype)) || !aligned(d->labels, 4) || !aligned(row_scale, stat) ||
        !aligned(log_sums_in, stat) || !aligned(loss, stat) || !aligned(log_sums_out, stat)) {
        fail("distill: a tensor is not aligned to its type");
        return PCU_ERR_ARGUMENT;
    }
    const Range student{l->data, logits_bytes(*l)};
    const Range values{d->teacher_values, l->rows * d->k * logit_size(d->teacher_dtype)},
        indices{d->teacher_indices, l->rows * d->k * 4}, whole{d->teacher_log_sum, l->rows * stat_size(d->teacher_dtype)},
        labels{d->labels, l->rows * 4}, scale{row_scale, l->rows * stat}, sums{log_sums_in, l->rows * 2 * stat};
    const Range out_loss{loss, l->rows * stat}, out_sums{log_sums_out, l->rows * 2 * stat},
        out_grad{grad, strided_bytes(l->rows, grad_cols, grad_stride, size)};
    // A gradient in the logits' place, row for row, is read before it is written.
    const bool in_place = grad == l->data && grad_stride == l->stride;
    if ((!in_place && overlaps_any(out_grad, {student})) ||
        overlaps_any(out_grad, {values, indices, whole, labels, scale, sums, out_loss, out_sums}) ||
        overlaps_any(out_loss, {student, values, indices, whole, labels, scale, sums, out_sums}) ||
        overlaps_any(out_sums, {student, values, indices, whole, labels, scale})) {
        fail("distill: an output overlaps another tensor");
        return PCU_ERR_ARGUMENT;
    }
    unsigned long long *word;
    if ((st = add_node(NodeInfo{Prim::Checked, l->rows * (d->k + 1), 0}, &word)))
        return st;
    DistillArgs g;
    g.logits = l->data;
    g.dtype = (int)l->dtype;
    g.rows = l->rows;
    g.stride = l->stride;
    g.vocab = (uint32_t)l->vocab;
    g.k = d->k;
    g.teacher_values = d->teacher_values;
    g.teacher_dtype = (int)d->teacher_dtype;
    g.teacher_indices = d->teacher_indices;
    g.teacher_log_sum = d->teacher_log_sum;
    g.teacher_log_sum_f64 = d->teacher_dtype == PCU_F64;
    g.labels = d->labels;
    g.temperature = d->temperature;
    g.distill_weight = d->distill_weight;
    g.label_weight = d->label_weight;
    g.row_scale = row_scale;
    g.log_sums_in = log_sums_in;
    g.log_sums_out = log_sums_out;
    g.loss = loss;
    g.grad = grad;
    g.grad_stride = grad_stride;
    g.grad_cols = (uint32_t)grad_cols;
    g.fault = word;
    g.gate = gate_for(word);
    void *sc = nullptr;
    const size_t need = distill_scratch_bytes(g);
    if (need && (st = scratch(logits_scratch, need, false, &sc)))
        return st;
    if ((st = open_words()))
        return st;
    ProgramClose close;
    if (implicit_program && nodes.size() == 1)
        close_next = true; // a call of its own: its kernel ends the program
    if ((st = take_close(&close)))
        return st;
    bool closed = false;
    hipEvent_t t = timer_start(stream);
    st = hip(launch_distill(stream, g, sc, close, &closed), "distill launch");
    timer_stop(PCU_KERNEL_DISTILL, t, stream);
    if (!st && closed)
        closed_seq = ++pub_seq;
    return st;
}

pcu_status Ctx::op_sample(const pcu_logits *l, const pcu_sampling *p, int32_t *tokens, float *log_prob)
{
    pcu_status st = check_logits(this, "sample", l);
    if (st)
        return st;
    if (!p || (l->rows && (!p->uniform || !tokens))) {
        fail("sample: invalid argument");
        return PCU_ERR_ARGUMENT;
    }
    for (const void *x : {(const void *)p->uniform, (const void *)p->temperature, (const void *)p->top_k,
                          (const void *)p->top_p, (const void *)p->min_p, (const void *)tokens, (const void *)log_prob})
        if (!aligned(x, 4)) {
            fail("sample: a tensor is not aligned to its type");
            return PCU_ERR_ARGUMENT;
        }
    const uint64_t b = l->rows * 4;
    const Range logits{l->data, logits_bytes(*l)}, u{p->uniform, b}, t{p->temperature, b}, tk{p->top_k, b},
        tp{p->top_p, b}, mp{p->min_p, b}, out{tokens, b}, lp{log_prob, b};
    if (overlaps_any(out, {logits, u, t, tk, tp, mp, lp}) || overlaps_any(lp, {logits, u, t, tk, tp, mp})) {
        fail("sample: an output overlaps another tensor");
        return PCU_ERR_ARGUMENT;
    }
    // Settings that hold for every row are checked here (a NaN fails every comparison).
    if ((!p->temperature && !(p->temperature_value >= 0 && std::isfinite(p->temperature_value))) ||
        (!p->top_p && !(p->top_p_value >= 0 && p->top_p_value <= 1)) ||
        (!p->min_p && !(p->min_p_value >= 0 && p->min_p_value <= 1))) {
        fail("sample: a setting is out of its range");
        return PCU_ERR_ARGUMENT;
    }
    unsigned long long *word;
    if ((st = add_node(NodeInfo{Prim::Checked, l->rows, 0}, &word)))
        return st;
    SampleArgs g;
    g.logits = l->data;
    g.dtype = (int)l->dtype;
    g.rows = l->rows;
    g.stride = l->stride;
    g.vocab = (uint32_t)l->vocab;
    g.uniform = p->uniform;
    g.temperature = p->temperature;
    g.top_k = p->top_k;
    g.top_p = p->top_p;
    g.min_p = p->min_p;
    g.temperature_all = p->temperature_value;
    g.top_k_all = p->top_k_value;
    g.top_p_all = p->top_p_value;
    g.min_p_all = p->min_p_value;
    g.tokens = tokens;
    g.log_prob = log_prob;
    g.fault = word;
    g.gate = gate_for(word);
    void *sc = nullptr, *state = nullptr;
    const size_t need = sample_scratch_bytes(g);
    if (need && (st = scratch(logits_scratch, need, false, &sc)))
        return st;
    if (need && (st = scratch(sample_state, sample_state_bytes(), false, &state)))
        return st;
    if ((st = open_words()))
        return st;
    ProgramClose close;
    if (implicit_program && nodes.size() == 1)
        close_next = true; // a call of its own: its last kernel ends the program
    if ((st = take_close(&close)))
        return st;
    bool closed = false;
    hipEvent_t ev = timer_start(stream);
    if (need && !sample_state_zero) {
        if ((st = hip(launch_fill_u64(stream, static_cast<unsigned long long *>(state), sample_state_bytes() / 8, 0),
                      "sample state")))
            return st;
        sample_state_zero = true;
    }
    st = hip(launch_sample(stream, g, sc, state, close, &closed), "sample launch");
    if (st)
        sample_state_zero = false;
    timer_stop(PCU_KERNEL_SAMPLE, ev, stream);
    if (!st && closed)
        closed_seq = ++pub_seq;
    return st;
}

} // namespace pcu

using pcu::Ctx;

extern "C" {

pcu_status pcu_native_top_logits(pcu_ctx *ctx, const pcu_logits *logits, uint32_t k, double temperature,
                                 void *values, int32_t *indices, void *log_sum)
{
    pcu_status st;
    Ctx *c = pcu::enter(ctx, &st);
    if (!c)
        return st;
    return c->finish_op(c->op_top_logits(logits, k, temperature, values, indices, log_sum), nullptr);
}

pcu_status pcu_native_distill_loss(pcu_ctx *ctx, const pcu_logits *student, const pcu_distill *distill,
                                   void *loss, void *log_sums, pcu_fault *fault)
{
    pcu_status st;
    Ctx *c = pcu::enter(ctx, &st);
    if (!c)
        return st;
    return c->finish_op(c->op_distill(Ctx::Distill::Loss, student, distill, nullptr, nullptr, loss, log_sums,
                                      nullptr, 0, 0), fault);
}

pcu_status pcu_native_distill_backward(pcu_ctx *ctx, const pcu_logits *student, const pcu_distill *distill,
                                       const void *log_sums, const void *row_scale, void *gradient,
                                       uint64_t gradient_cols, uint64_t gradient_stride, pcu_fault *fault)
{
    pcu_status st;
    Ctx *c = pcu::enter(ctx, &st);
    if (!c)
        return st;
    return c->finish_op(c->op_distill(Ctx::Distill::Backward, student, distill, log_sums, row_scale, nullptr,
                                      nullptr, gradient, gradient_cols, gradient_stride), fault);
}

pcu_status pcu_native_distill_step(pcu_ctx *ctx, const pcu_logits *student, const pcu_distill *distill,
                                   const void *row_scale, void *loss, void *gradient, uint64_t gradient_cols,
                                   uint64_t gradient_stride, pcu_fault *fault)
{
    pcu_status st;
    Ctx *c = pcu::enter(ctx, &st);
    if (!c)
        return st;
    return c->finish_op(c->op_distill(Ctx::Distill::Step, student, distill, nullptr, row_scale, loss, nullptr,
                                      gradient, gradient_cols, gradient_stride), fault);
}

pcu_status pcu_native_sample(pcu_ctx *ctx, const pcu_logits *logits, const pcu_sampling *sampling,
                             int32_t *tokens, float *log_prob, pcu_fault *fault)
{
    pcu_status st;
    Ctx *c = pcu::enter(ctx, &st);
    if (!c)
        return st;
    return c->finish_op(c->op_sample(logits, sampling, tokens, log_prob), fault);
}

} // extern "C"
