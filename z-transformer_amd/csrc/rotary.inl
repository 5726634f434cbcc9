// Entry points of rotary positions in general (include/zt_attn.h): included by zt_attn.cpp behind paged.inl, inside
// its extern "C" block.

int zt_rope_frequencies(double *freq, int rot_dim, double theta, int scaling, double factor, double low, double high,
                        double context) {
    if (!freq || rot_dim < 2 || rot_dim > kMaxDim || rot_dim % 2 != 0) {
        fprintf(stderr, "zt_rope: %d rotated columns have no frequencies here. They must be even, in [2, %d].\n", rot_dim,
                kMaxDim);
        return 1;
    }
    if (!(theta > 0.0) || !std::isfinite(theta)) {
        fprintf(stderr, "zt_rope: theta %g is not usable.\n", theta);
        return 1;
    }
    const bool base = scaling == ZT_ROPE_BASE, turns = scaling == ZT_ROPE_TURNS;
    if (scaling < ZT_ROPE_PLAIN || scaling > ZT_ROPE_TURNS ||
        (scaling != ZT_ROPE_PLAIN && (!(factor > 0.0) || !std::isfinite(factor))) || (base && rot_dim < 4) ||
        (turns && (!(high > low) || !std::isfinite(high - low) || !(context > 0.0) || !std::isfinite(context)))) {
        fprintf(stderr, "zt_rope: scaling %d by %g between %g and %g turns of %g positions is not usable.\n", scaling, factor,
                low, high, context);
        return 1;
    }
    const double b = base ? theta * std::pow(factor, rot_dim / (rot_dim - 2.0)) : theta;
    double got[kMaxDim / 2];
    for (int i = 0; i < rot_dim / 2; ++i) {
        const double f = std::pow(b, -2.0 * i / rot_dim);
        double by = scaling == ZT_ROPE_LINEAR ? 1.0 / factor : 1.0;
        if (turns) {
            const double r = context * f / 6.283185307179586476925286766559;
            const double part = std::min(1.0, std::max(0.0, (r - low) / (high - low)));
            by = part + (1.0 - part) / factor;
        }
        got[i] = f * by;
        if (!(b > 0.0) || !std::isfinite(b) || !std::isfinite(got[i])) {
            fprintf(stderr, "zt_rope: frequency %d of theta %g, scaled by %g, is beyond 64 bits.\n", i, theta, factor);
            return 1;
        }
    }
    std::copy(got, got + rot_dim / 2, freq);
    return 0;
}

// What a call turns, into its arguments; 0 when usable.
static int turn_check(const double *freq, int rot_dim, int interleaved, double amplitude, int dim, TurnArgs *a) {
    if (rot_dim < 2 || rot_dim > dim || rot_dim % 2 != 0) {
        fprintf(stderr, "zt_rope: %d rotated columns of %d are not usable. They must be even and within the head.\n", rot_dim,
                dim);
        return 1;
    }
    if (interleaved != 0 && interleaved != 1) {
        fprintf(stderr, "zt_rope: interleaved is 0 or 1, not %d.\n", interleaved);
        return 1;
    }
    if (!freq || !std::isfinite(amplitude)) {
        fprintf(stderr, "zt_rope: the host frequencies and a finite amplitude are needed.\n");
        return 1;
    }
    for (int i = 0; i < rot_dim / 2; ++i) {
        if (!std::isfinite(freq[i])) {
            fprintf(stderr, "zt_rope: frequency %d is %g.\n", i, freq[i]);
            return 1;
        }
        a->freq[i] = freq[i];
    }
    a->dim = dim; a->rot = rot_dim;
    a->amplitude = a->sine = amplitude;
    return 0;
}

// Whole vectors: of four or two pairs' halves, or of two neighbouring pairs.
static const char *turn_kind(int dim, int rot_dim, int interleaved) {
    if (interleaved) return dim % 4 == 0 && rot_dim % 4 == 0 ? "inter2" : "inter1";
    return dim % 4 == 0 && rot_dim % 8 == 0 ? "half4" : rot_dim % 4 == 0 ? "half2" : "half1";
}

// Launches `name` for rows a.row0 .. a.row0 + rows - 1, `units` of work in each: few rows are cut into parts.
extern "C++" {
namespace {
template <class Args>
int turn_launch(DeviceState *st, const char *name, Args &x, TurnArgs &a, long long rows, long long units,
                hipStream_t stream) {
    const long long most = 0xFFFFFFFFll / kThreads;
    const int row0 = a.row0;
    for (long long r = 0; r < rows; r += most) {
        a.row0 = (int)(row0 + r);
        a.rows = (int)std::min(most, rows - r);
        a.slices = (int)std::max(1LL, std::min(1024LL / a.rows, (units + kThreads - 1) / kThreads));
        if (launch(st, name, (unsigned)a.rows * (unsigned)a.slices, x, stream)) return 1;
    }
    return 0;
}
}  // namespace
}  // extern "C++"

static int rope_at(const float *q, const float *k, float *q_out, float *k_out, const int *pos, const double *freq, int rows,
                   int n_heads, int n_kv_heads, int head_dim, int rot_dim, int interleaved, double amplitude, bool back,
                   hipStream_t stream) {
    if (head_dim < 2 || head_dim > kMaxDim || head_dim % 2 != 0) {
        fprintf(stderr, "zt_rope: head_dim %d is odd or outside [2, %d].\n", head_dim, kMaxDim);
        return 1;
    }
    if (rows < 0 || n_heads < 0 || n_kv_heads < 0 || n_heads > 65535 || n_kv_heads > 65535) {
        fprintf(stderr, "zt_rope: %d rows of %d + %d heads are not launchable.\n", rows, n_heads, n_kv_heads);
        return 1;
    }
    TurnArgs a{};
    if (turn_check(freq, rot_dim, interleaved, amplitude, head_dim, &a)) return 1;
    if (back) a.sine = -a.sine;
    if (rows == 0 || n_heads + n_kv_heads == 0) return 0;
    if (!pos || (n_heads > 0 && (!q || !q_out)) || (n_kv_heads > 0 && (!k || !k_out))) {
        fprintf(stderr, "zt_rope: a null tensor pointer is not launchable.\n");
        return 1;
    }
    if (!rows_aligned(head_dim, {q, k, q_out, k_out})) return 1;
    DeviceState *st = device_state();
    if (!st) {
        fprintf(stderr, "zt_rope: no usable gfx950 device or code object.\n");
        return 1;
    }
    a.q = n_heads ? q : nullptr; a.k = n_kv_heads ? k : nullptr;
    a.q_out = n_heads ? q_out : nullptr; a.k_out = n_kv_heads ? k_out : nullptr;
    a.pos = pos; a.H = n_heads; a.Hkv = n_kv_heads;
    char name[64];
    snprintf(name, sizeof name, "zt_turn_%s", turn_kind(head_dim, rot_dim, interleaved));
    return turn_launch(st, name, a, a, rows, (n_heads + n_kv_heads) * (head_dim / 8 + 1LL), stream);
}

int zt_rope_at_forward(const float *q, const float *k, float *q_out, float *k_out, const int *pos, const double *freq,
                       int rows, int n_heads, int n_kv_heads, int head_dim, int rot_dim, int interleaved, double amplitude,
                       hipStream_t stream) {
    return rope_at(q, k, q_out, k_out, pos, freq, rows, n_heads, n_kv_heads, head_dim, rot_dim, interleaved, amplitude, false,
                   stream);
}

int zt_rope_at_backward(const float *dq, const float *dk, float *dq_out, float *dk_out, const int *pos, const double *freq,
                        int rows, int n_heads, int n_kv_heads, int head_dim, int rot_dim, int interleaved,
                        double amplitude, hipStream_t stream) {
    return rope_at(dq, dk, dq_out, dk_out, pos, freq, rows, n_heads, n_kv_heads, head_dim, rot_dim, interleaved, amplitude,
                   true, stream);
}

int zt_paged_append_at(const float *q, const float *k_new, const float *v_new, float *q_out, float *k_pages,
                       float *v_pages, const int *table, float *w, const int *pos, const double *freq, const int *q_start,
                       const int *n_rows, int B, int n_pages, int page_size, int table_stride, int w_stride, int n_heads,
                       int n_kv_heads, int dim, int rot_dim, int interleaved, double amplitude, hipStream_t stream) {
    if (paged_check("paged_append_at", n_rows, B, n_pages, page_size, table_stride)) return 1;
    if (!zt_attn_dim_ok(dim)) return refuse_dim(dim);
    if (check_group(n_heads, n_kv_heads)) return 1;
    if (paged_tokens_check("paged_append_at", q_start, n_rows, B, n_heads)) return 1;
    if (w && paged_weights_check("paged_append_at", n_rows, B, w_stride)) return 1;
    TurnPagedArgs a{};
    if (turn_check(freq, rot_dim, interleaved, amplitude, dim, &a.turn)) return 1;
    const bool any = q_start[B] > q_start[0];
    if (!k_pages || !v_pages || !table || (any && (!k_new || !v_new || !pos)) || !q != !q_out) {
        fprintf(stderr, "zt_attn: a null tensor pointer is not launchable.\n");
        return 1;
    }
    if (!rows_aligned(dim, {q, k_new, v_new, q_out, k_pages, v_pages})) return 1;
    DeviceState *st = require_device();
    if (!st) return 1;
    a.pool = page_pool(k_pages, v_pages, table, n_pages, page_size, table_stride);
    a.v_new = v_new; a.w = w; a.w_stride = w_stride;
    a.turn.q = q; a.turn.q_out = q_out; a.turn.k = k_new; a.turn.pos = pos;
    a.turn.H = n_heads; a.turn.Hkv = n_kv_heads;
    char name[64];
    snprintf(name, sizeof name, "zt_turn_paged_%s", turn_kind(dim, rot_dim, interleaved));
    for (int b = 0; b < B;) {
        a.ns = 0;
        const int first = q_start[b];
        for (; b < B && a.ns < ZT_PAGED_MAXB; ++b) {
            const int q_len = q_start[b + 1] - q_start[b];
            if (q_len == 0) continue;
            const int i = a.ns++;
            a.b[i] = b; a.q0[i] = q_start[b]; a.first[i] = n_rows[b] - q_len;
        }
        a.turn.row0 = first;
        const long long units = ((q ? n_heads : 0) + 2LL * n_kv_heads) * (dim / 8 + 1);
        if (turn_launch(st, name, a, a.turn, q_start[b] - first, units, stream)) return 1;
    }
    return 0;
}
