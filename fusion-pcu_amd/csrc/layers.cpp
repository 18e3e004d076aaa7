// The operators around a model's products behind the C ABI: argument checks, scratch and launches.
#include "pcu_checks.hpp"

namespace pcu {

static_assert(kLogitF32 == PCU_F32 && kLogitF64 == PCU_F64 && kLogitBf16 == PCU_BF16 && kLogitF16 == PCU_F16,
              "one numbering");

static Range rows_range(const pcu_rows &r)
{
    return Range{r.data, strided_bytes(r.rows, r.cols, r.stride, logit_size(r.dtype))};
}

static pcu_status check_rows(Ctx *c, const char *what, const pcu_rows *r)
{
    if (!r || r->dtype > PCU_F16 || (r->rows && r->cols && !r->data) || !aligned(r->data, logit_size(r->dtype))) {
        c->fail("%s: invalid rows", what);
        return PCU_ERR_ARGUMENT;
    }
    if (r->cols > PCU_ROWS_MAX_COLS || r->rows > PCU_ROWS_MAX_ROWS || r->stride > PCU_ROWS_MAX_ROWS || r->stride < r->cols) {
        c->fail("%s: %llu rows of %llu values, stride %llu: beyond the limits", what, (unsigned long long)r->rows,
                (unsigned long long)r->cols, (unsigned long long)r->stride);
        return PCU_ERR_SHAPE;
    }
    return PCU_OK;
}

// An output (or a second input) of `rows` rows like those of `like`.
static pcu_status check_like(Ctx *c, const char *what, const void *p, uint64_t rows, uint64_t cols, uint64_t stride, uint64_t size)
{
    if ((rows && cols && !p) || !aligned(p, size)) {
        c->fail("%s: invalid rows", what);
        return PCU_ERR_ARGUMENT;
    }
    if (stride < cols || stride > PCU_ROWS_MAX_ROWS) {
        c->fail("%s: stride %llu for %llu values", what, (unsigned long long)stride, (unsigned long long)cols);
        return PCU_ERR_SHAPE;
    }
    return PCU_OK;
}

pcu_status Ctx::op_embedding(const pcu_rows *table, const int32_t *tokens, uint64_t count, double scale, void *out,
                             uint64_t out_stride)
{
    pcu_status st = check_rows(this, "embedding", table);
    if (st)
        return st;
    if (table->rows > PCU_TABLE_MAX_ROWS || count > PCU_ROWS_MAX_ROWS) {
        fail("embedding: a table of %llu rows, %llu tokens: beyond the limits", (unsigned long long)table->rows,
             (unsigned long long)count);
        return PCU_ERR_SHAPE;
    }
    const uint64_t size = logit_size(table->dtype);
    if ((st = check_like(this, "embedding: out", out, count, table->cols, out_stride, size)))
        return st;
    if ((count && !tokens) || !aligned(tokens, 4) || !valid_weight(table->dtype, scale)) {
        fail("embedding: invalid argument");
        return PCU_ERR_ARGUMENT;
    }
    if (overlaps_any(Range{out, strided_bytes(count, table->cols, out_stride, size)},
                     {rows_range(*table), Range{tokens, count * 4}})) {
        fail("embedding: an output overlaps another tensor");
        return PCU_ERR_ARGUMENT;
    }
    unsigned long long *word;
    if ((st = add_node(NodeInfo{Prim::Checked, count, 0}, &word)))
        return st;
    EmbedArgs g;
    g.table = table->data;
    g.dtype = (int)table->dtype;
    g.vocab = (uint32_t)table->rows;
    g.width = (uint32_t)table->cols;
    g.table_stride = table->stride;
    g.tokens = tokens;
    g.rows = count;
    g.scale = scale;
    g.out = out;
    g.out_stride = out_stride;
    g.fault = word;
    g.gate = gate_for(word);
    if ((st = open_words()))
        return st;
    ProgramClose close;
    if (implicit_program && nodes.size() == 1)
        close_next = true; // a call of its own: its kernel ends the program
    if ((st = take_close(&close)))
        return st;
    bool closed = false;
    hipEvent_t t = timer_start(stream);
    st = hip(launch_embed(stream, g, close, &closed), "embedding launch");
    timer_stop(PCU_KERNEL_EMBEDDING, t, stream);
    if (!st && closed)
        closed_seq = ++pub_seq;
    return st;
}

pcu_status Ctx::op_embedding_backward(const pcu_rows *gradient, const int32_t *tokens, uint64_t table_rows, double scale,
                                      const void *base, uint64_t base_stride, void *out, uint64_t out_stride)
{
    pcu_status st = check_rows(this, "embedding gradient", gradient);
    if (st)
        return st;
    const uint64_t size = logit_size(gradient->dtype), cols = gradient->cols;
    if (table_rows > PCU_TABLE_MAX_ROWS || gradient->rows * ((cols * size + 1023) / 1024) > 1ull << 28) {
        fail("embedding gradient: %llu x %llu for a table of %llu rows: beyond the limits", (unsigned long long)gradient->rows,
             (unsigned long long)cols, (unsigned long long)table_rows);
        return PCU_ERR_SHAPE;
    }
    if ((st = check_like(this, "embedding gradient: out", out, table_rows, cols, out_stride, size)) ||
        (base && (st = check_like(this, "embedding gradient: base", base, table_rows, cols, base_stride, size))))
        return st;
    if ((gradient->rows && !tokens) || !aligned(tokens, 4) || !valid_weight(gradient->dtype, scale)) {
        fail("embedding gradient: invalid argument");
        return PCU_ERR_ARGUMENT;
    }
    const Range o{out, strided_bytes(table_rows, cols, out_stride, size)};
    const bool in_place = base == out && base_stride == out_stride;
    if (overlaps_any(o, {rows_range(*gradient), Range{tokens, gradient->rows * 4}}) ||
        (base && !in_place && overlaps_any(o, {Range{base, strided_bytes(table_rows, cols, base_stride, size)}}))) {
        fail("embedding gradient: an output overlaps another tensor");
        return PCU_ERR_ARGUMENT;
    }
    unsigned long long *word;
    if ((st = add_node(NodeInfo{Prim::Checked, gradient->rows, 0}, &word)))
        return st;
    EmbedBackArgs g;
    g.gradient = gradient->data;
    g.dtype = (int)gradient->dtype;
    g.vocab = (uint32_t)table_rows;
    g.width = (uint32_t)cols;
    g.rows = gradient->rows;
    g.gradient_stride = gradient->stride;
    g.tokens = tokens;
    g.scale = scale;
    g.base = base;
    g.base_stride = base_stride;
    g.out = out;
    g.out_stride = out_stride;
    g.fault = word;
    g.gate = gate_for(word);
    void *sc = nullptr;
    const size_t need = embed_back_scratch_bytes(g);
    if (need && (st = scratch(layer_scratch, need, false, &sc)))
        return st;
    if ((st = open_words()))
        return st;
    ProgramClose close;
    if (implicit_program && nodes.size() == 1)
        close_next = true; // a call of its own: its last kernel ends the program
    if ((st = take_close(&close)))
        return st;
    bool closed = false;
    hipEvent_t t = timer_start(stream);
    st = hip(launch_embed_back(stream, g, sc, close, &closed), "embedding gradient launch");
    timer_stop(PCU_KERNEL_EMBEDDING, t, stream);
    if (!st && closed)
        closed_seq = ++pub_seq;
    return st;
}

static bool valid_weight_dtype(uint32_t dtype, int weight_dtype)
{
    return weight_dtype == (int)dtype || (weight_dtype == PCU_F32 && (dtype == PCU_BF16 || dtype == PCU_F16));
}

pcu_status Ctx::op_layer_norm(const pcu_rows *x, const void *weight, const void *bias, int weight_dtype, double eps,
                              void *out, uint64_t out_stride, void *stats)
{
    pcu_status st = check_rows(this, "layer_norm", x);
    if (st)
        return st;
    const uint64_t size = logit_size(x->dtype);
    if ((st = check_like(this, "layer_norm: out", out, x->rows, x->cols, out_stride, size)))
        return st;
    if (!valid_weight_dtype(x->dtype, weight_dtype) || !(eps >= 0) || !valid_weight(x->dtype, eps) ||
        !aligned(weight, logit_size(weight_dtype)) || !aligned(bias, logit_size(weight_dtype)) ||
        !aligned(stats, stat_size(x->dtype))) {
        fail("layer_norm: invalid argument");
        return PCU_ERR_ARGUMENT;
    }
    const uint64_t wb = x->cols * logit_size(weight_dtype);
    const Range o{out, strided_bytes(x->rows, x->cols, out_stride, size)}, s{stats, x->rows * 2 * stat_size(x->dtype)},
        w{weight, wb}, b{bias, wb};
    const bool in_place = out == x->data && out_stride == x->stride;
    if ((!in_place && overlaps_any(o, {rows_range(*x)})) || overlaps_any(o, {w, b, s}) ||
        overlaps_any(s, {rows_range(*x), w, b})) {
        fail("layer_norm: an output overlaps another tensor");
        return PCU_ERR_ARGUMENT;
    }
    unsigned long long *word;
    if ((st = add_node(NodeInfo{Prim::Native, x->rows, 0}, &word)))
        return st;
    NormArgs g;
    g.x = x->data;
    g.dtype = (int)x->dtype;
    g.weight_dtype = weight_dtype;
    g.rows = x->rows;
    g.stride = x->stride;
    g.width = (uint32_t)x->cols;
    g.weight = weight;
    g.bias = bias;
    g.eps = eps;
    g.out = out;
    g.out_stride = out_stride;
    g.stats = stats;
    g.gate = gate_for(word);
    if ((st = open_words()))
        return st;
    ProgramClose close;
    if (implicit_program && nodes.size() == 1)
        close_next = true; // a call of its own: its kernel ends the program
    if ((st = take_close(&close)))
        return st;
    bool closed = false;
    hipEvent_t t = timer_start(stream);
    st = hip(launch_norm(stream, g, close, &closed), "layer_norm launch");
    timer_stop(PCU_KERNEL_LAYER_NORM, t, stream);
    if (!st && closed)
        closed_seq = ++pub_seq;
    return st;
}

pcu_status Ctx::op_layer_norm_backward(const pcu_rows *x, const void *stats, const void *gradient,
                                       uint64_t gradient_stride, const void *weight, int weight_dtype, void *x_gradient,
                                       uint64_t x_gradient_stride, void *weight_gradient, void *bias_gradient)
{
    pcu_status st = check_rows(this, "layer_norm gradient", x);
    if (st)
        return st;
    const uint64_t size = logit_size(x->dtype), stat = stat_size(x->dtype);
    if ((st = check_like(this, "layer_norm gradient: gradient", gradient, x->rows, x->cols, gradient_stride, size)) ||
        (x_gradient &&
         (st = check_like(this, "layer_norm gradient: x_gradient", x_gradient, x->rows, x->cols, x_gradient_stride, size))))
        return st;
    if (!valid_weight_dtype(x->dtype, weight_dtype)) {
        fail("layer_norm gradient: invalid weight type");
        return PCU_ERR_ARGUMENT;
    }
    const uint64_t ws = logit_size(weight_dtype);
    if ((x->rows && x->cols && !stats) || !aligned(stats, stat) || !aligned(weight, ws) || !aligned(weight_gradient, ws) ||
        !aligned(bias_gradient, ws)) {
        fail("layer_norm gradient: invalid argument");
        return PCU_ERR_ARGUMENT;
    }
    const Range rx = rows_range(*x), s{stats, x->rows * 2 * stat}, w{weight, x->cols * ws},
        dy{gradient, strided_bytes(x->rows, x->cols, gradient_stride, size)},
        dx{x_gradient, strided_bytes(x->rows, x->cols, x_gradient_stride, size)}, dw{weight_gradient, x->cols * ws},
        db{bias_gradient, x->cols * ws};
    const bool on_x = x_gradient == x->data && x_gradient_stride == x->stride;
    const bool on_dy = x_gradient == gradient && x_gradient_stride == gradient_stride;
    if ((!on_x && overlaps_any(dx, {rx})) || (!on_dy && overlaps_any(dx, {dy})) || overlaps_any(dx, {s, w, dw, db}) ||
        overlaps_any(dw, {rx, dy, s, w, db}) || overlaps_any(db, {rx, dy, s, w})) {
        fail("layer_norm gradient: an output overlaps another tensor");
        return PCU_ERR_ARGUMENT;
    }
    unsigned long long *word;
    if ((st = add_node(NodeInfo{Prim::Native, x->rows, 0}, &word)))
        return st;
    NormBackArgs g;
    g.x = x->data;
    g.dtype = (int)x->dtype;
    g.weight_dtype = weight_dtype;
    g.rows = x->rows;
    g.stride = x->stride;
    g.width = (uint32_t)x->cols;
    g.stats = stats;
    g.gradient = gradient;
    g.gradient_stride = gradient_stride;
    g.weight = weight;
    g.x_gradient = x_gradient;
    g.x_gradient_stride = x_gradient_stride;
    g.weight_gradient = weight_gradient;
    g.bias_gradient = bias_gradient;
    g.gate = gate_for(word);
    void *sc = nullptr;
    const size_t need = norm_back_scratch_bytes(g);
    if (need && (st = scratch(layer_scratch, need, false, &sc)))
        return st;
    if ((st = open_words()))
        return st;
    ProgramClose close;
    if (implicit_program && nodes.size() == 1)
        close_next = true; // a call of its own: its last kernel ends the program
    if ((st = take_close(&close)))
        return st;
    bool closed = false;
    hipEvent_t t = timer_start(stream);
    st = hip(launch_norm_back(stream, g, sc, close, &closed), "layer_norm gradient launch");
    timer_stop(PCU_KERNEL_LAYER_NORM, t, stream);
    if (!st && closed)
        closed_seq = ++pub_seq;
    return st;
}

pcu_status Ctx::op_cross_entropy(const pcu_rows *features, const pcu_rows *weights, bool loss, EntropyArgs g)
{
    pcu_status st = check_rows(this, "cross_entropy: features", features);
    if (st || (st = check_rows(this, "cross_entropy: weights", weights)))
        return st;
    if (features->dtype != weights->dtype) {
        fail("cross_entropy: features and weights of different types");
        return PCU_ERR_ARGUMENT;
    }
    if (features->dtype == PCU_F64) {
        fail("cross_entropy: F64 features are not admitted");
        return PCU_ERR_UNSUPPORTED;
    }
    const uint64_t rows = features->rows, width = features->cols, size = logit_size(features->dtype);
    constexpr uint64_t kMost = 1ull << 37; // of any two of the sizes: the launches' grids
    if (width != weights->cols || width < 1 || width > PCU_ENTROPY_MAX_WIDTH || rows > PCU_ENTROPY_MAX_ROWS ||
        weights->rows > PCU_TABLE_MAX_ROWS || rows * weights->rows > kMost || rows * width > kMost || width * weights->rows > kMost) {
        fail("cross_entropy: %llu x %llu features, %llu x %llu weights", (unsigned long long)rows, (unsigned long long)width,
             (unsigned long long)weights->rows, (unsigned long long)weights->cols);
        return PCU_ERR_SHAPE;
    }
    if (g.weight_gradient && (g.weight_gradient_rows < weights->rows || g.weight_gradient_rows > PCU_TABLE_MAX_ROWS)) {
        fail("cross_entropy: a gradient of %llu rows for %llu", (unsigned long long)g.weight_gradient_rows,
             (unsigned long long)weights->rows);
        return PCU_ERR_SHAPE;
    }
    if ((g.feature_gradient && (st = check_like(this, "cross_entropy: feature gradient", g.feature_gradient, rows, width,
                                                g.feature_gradient_stride, size))) ||
        (g.weight_gradient && (st = check_like(this, "cross_entropy: weight gradient", g.weight_gradient, g.weight_gradient_rows,
                                               width, g.weight_gradient_stride, size))))
        return st;
    if ((rows && (!g.labels || (loss ? !g.loss : !g.log_sum_in))) || !aligned(g.labels, 4) || !aligned(g.log_sum_in, 4) ||
        !aligned(g.row_scale, 4) || !aligned(g.loss, 4) || !aligned(g.log_sum_out, 4)) {
        fail("cross_entropy: invalid argument");
        return PCU_ERR_ARGUMENT;
    }
    const Range x = rows_range(*features), w = rows_range(*weights), labels{g.labels, rows * 4}, sums{g.log_sum_in, rows * 4},
        scale{g.row_scale, rows * 4};
    const Range l{g.loss, rows * 4}, ls{g.log_sum_out, rows * 4},
        dx{g.feature_gradient, strided_bytes(rows, width, g.feature_gradient_stride, size)},
        dw{g.weight_gradient, strided_bytes(g.weight_gradient_rows, width, g.weight_gradient_stride, size)};
    if (overlaps_any(l, {x, w, labels, sums, scale, ls, dx, dw}) || overlaps_any(ls, {x, w, labels, sums, scale, dx, dw}) ||
        overlaps_any(dx, {x, w, labels, sums, scale, dw}) || overlaps_any(dw, {x, w, labels, sums, scale})) {
        fail("cross_entropy: an output overlaps another tensor");
        return PCU_ERR_ARGUMENT;
    }
    unsigned long long *word;
    if ((st = add_node(NodeInfo{Prim::Checked, rows, 0}, &word)))
        return st;
    g.features = features->data;
    g.dtype = (int)features->dtype;
    g.rows = rows;
    g.feature_stride = features->stride;
    g.width = (uint32_t)width;
    g.vocab = (uint32_t)weights->rows;
    g.weights = weights->data;
    g.weight_stride = weights->stride;
    g.fault = word;
    g.gate = gate_for(word);
    void *sc = nullptr;
    if ((st = scratch(layer_scratch, entropy_scratch_bytes(g), false, &sc)))
        return st;
    if ((st = open_words()))
        return st;
    ProgramClose close;
    if (implicit_program && nodes.size() == 1)
        close_next = true; // a call of its own: its last kernel ends the program
    if ((st = take_close(&close)))
        return st;
    bool closed = false;
    hipEvent_t t = timer_start(stream);
    st = hip(launch_entropy(stream, g, sc, close, &closed), "cross_entropy launch");
    timer_stop(PCU_KERNEL_CROSS_ENTROPY, t, stream);
    if (!st && closed)
        closed_seq = ++pub_seq;
    return st;
}

} // namespace pcu

using pcu::Ctx;

extern "C" {

pcu_status pcu_native_embedding(pcu_ctx *ctx, const pcu_rows *table, const int32_t *tokens, uint64_t count, double scale,
                                void *out, uint64_t out_stride, pcu_fault *fault)
{
    pcu_status st;
    Ctx *c = pcu::enter(ctx, &st);
    if (!c)
        return st;
    return c->finish_op(c->op_embedding(table, tokens, count, scale, out, out_stride), fault);
}

pcu_status pcu_native_embedding_backward(pcu_ctx *ctx, const pcu_rows *gradient, const int32_t *tokens,
                                         uint64_t table_rows, double scale, const void *base, uint64_t base_stride,
                                         void *out, uint64_t out_stride, pcu_fault *fault)
{
    pcu_status st;
    Ctx *c = pcu::enter(ctx, &st);
    if (!c)
        return st;
    return c->finish_op(c->op_embedding_backward(gradient, tokens, table_rows, scale, base, base_stride, out, out_stride),
                        fault);
}

pcu_status pcu_native_layer_norm(pcu_ctx *ctx, const pcu_rows *x, const void *weight, const void *bias,
                                 pcu_dtype weight_dtype, double eps, void *out, uint64_t out_stride, void *stats)
{
    pcu_status st;
    Ctx *c = pcu::enter(ctx, &st);
    if (!c)
        return st;
    return c->finish_op(c->op_layer_norm(x, weight, bias, (int)weight_dtype, eps, out, out_stride, stats), nullptr);
}

pcu_status pcu_native_layer_norm_backward(pcu_ctx *ctx, const pcu_rows *x, const void *stats, const void *gradient,
                                          uint64_t gradient_stride, const void *weight, pcu_dtype weight_dtype,
                                          void *x_gradient, uint64_t x_gradient_stride, void *weight_gradient,
                                          void *bias_gradient)
{
    pcu_status st;
    Ctx *c = pcu::enter(ctx, &st);
    if (!c)
        return st;
    return c->finish_op(c->op_layer_norm_backward(x, stats, gradient, gradient_stride, weight, (int)weight_dtype, x_gradient,
                                                  x_gradient_stride, weight_gradient, bias_gradient), nullptr);
}

pcu_status pcu_native_cross_entropy_loss(pcu_ctx *ctx, const pcu_rows *features, const pcu_rows *weights,
                                         const int32_t *labels, float *loss, float *log_sum, pcu_fault *fault)
{
    pcu_status st;
    Ctx *c = pcu::enter(ctx, &st);
    if (!c)
        return st;
    pcu::EntropyArgs g;
    g.labels = labels;
    g.loss = loss;
    g.log_sum_out = log_sum;
    return c->finish_op(c->op_cross_entropy(features, weights, true, g), fault);
}

pcu_status pcu_native_cross_entropy_backward(pcu_ctx *ctx, const pcu_rows *features, const pcu_rows *weights,
                                             const int32_t *labels, const float *log_sum, const float *row_scale,
                                             void *feature_gradient, uint64_t feature_gradient_stride, void *weight_gradient,
                                             uint64_t weight_gradient_rows, uint64_t weight_gradient_stride, pcu_fault *fault)
{
    pcu_status st;
    Ctx *c = pcu::enter(ctx, &st);
    if (!c)
        return st;
    pcu::EntropyArgs g;
    g.labels = labels;
    g.log_sum_in = log_sum;
    g.row_scale = row_scale;
    g.feature_gradient = feature_gradient;
    g.feature_gradient_stride = feature_gradient_stride;
    g.weight_gradient = weight_gradient;
    g.weight_gradient_rows = weight_gradient_rows;
    g.weight_gradient_stride = weight_gradient_stride;
    return c->finish_op(c->op_cross_entropy(features, weights, false, g), fault);
}

pcu_status pcu_native_cross_entropy_step(pcu_ctx *ctx, const pcu_rows *features, const pcu_rows *weights,
                                         const int32_t *labels, const float *row_scale, float *loss, void *feature_gradient,
                                         uint64_t feature_gradient_stride, void *weight_gradient, uint64_t weight_gradient_rows,
                                         uint64_t weight_gradient_stride, pcu_fault *fault)
{
    pcu_status st;
    Ctx *c = pcu::enter(ctx, &st);
    if (!c)
        return st;
    pcu::EntropyArgs g;
    g.labels = labels;
    g.row_scale = row_scale;
    g.loss = loss;
    g.feature_gradient = feature_gradient;
    g.feature_gradient_stride = feature_gradient_stride;
    g.weight_gradient = weight_gradient;
    g.weight_gradient_rows = weight_gradient_rows;
    g.weight_gradient_stride = weight_gradient_stride;
    return c->finish_op(c->op_cross_entropy(features, weights, true, g), fault);
}

} // extern "C"
