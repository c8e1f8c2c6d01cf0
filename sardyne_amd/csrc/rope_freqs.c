/* Frequencies of scaled rotary positions, made on the host once per model. */
#include <math.h>

#include "sdy_internal.h"
#include "sdy_ops.h"

static const double TWO_PI = 6.283185307179586476925;

/* Plain: f_i = theta^(-2i / n_rot), as sdy_rope_table_host. Linear (position interpolation): f_i / factor.
 * YaRN: pairs that turn at least beta_fast times over the original context keep f_i, those that turn at most beta_slow
 * times take f_i / factor, a ramp over the pair's index between; cos and sin times attn_factor, or 0.1 ln factor + 1.
 * Llama3: pairs that turn high_freq times or more over the original context keep f_i, low_freq times or fewer take
 * f_i / factor, a ramp over the number of turns between. */
int sdy_rope_freqs(double *freq, float *mscale, int n_rot, float theta, const sdy_rope_scaling *sc) {
    if (!freq || !mscale) return sdy_fail(-1, "rope_freqs: freq and mscale are needed");
    if (n_rot < 0 || n_rot > 512 || n_rot % 2) return sdy_fail(-1, "rope_freqs: n_rot %d (even, 0..512)", n_rot);
    if (!(theta > 1.0f) || isinf(theta)) return sdy_fail(-1, "rope_freqs: theta %g (above 1)", (double)theta);
    const int kind = sc ? sc->kind : SDY_ROPE_PLAIN;
    if (kind < SDY_ROPE_PLAIN || kind > SDY_ROPE_LLAMA3) return sdy_fail(-1, "rope_freqs: scaling kind %d", kind);
    if (kind != SDY_ROPE_PLAIN && (!(sc->factor > 0.0f) || isinf(sc->factor)))
        return sdy_fail(-1, "rope_freqs: factor %g", (double)sc->factor);
    if (kind >= SDY_ROPE_YARN && sc->orig_ctx < 1) return sdy_fail(-1, "rope_freqs: orig_ctx %d", sc->orig_ctx);
    if (kind == SDY_ROPE_YARN && (!(sc->beta_slow > 0.0f) || !(sc->beta_fast >= sc->beta_slow) || !(sc->attn_factor >= 0.0f)))
        return sdy_fail(-1, "rope_freqs: beta_fast %g, beta_slow %g, attn_factor %g", (double)sc->beta_fast,
                        (double)sc->beta_slow, (double)sc->attn_factor);
    if (kind == SDY_ROPE_LLAMA3 && !(sc->high_freq > sc->low_freq))
        return sdy_fail(-1, "rope_freqs: low_freq %g below high_freq %g", (double)sc->low_freq, (double)sc->high_freq);
    double low = 0.0, high = 0.0;
    *mscale = 1.0f;
    if (kind == SDY_ROPE_YARN) {
        low = n_rot * log(sc->orig_ctx / (sc->beta_fast * TWO_PI)) / (2.0 * log(theta));
        high = n_rot * log(sc->orig_ctx / (sc->beta_slow * TWO_PI)) / (2.0 * log(theta));
        low = fmax(floor(low), 0.0);
        high = fmin(ceil(high), n_rot - 1.0);
        *mscale = sc->attn_factor > 0.0f ? sc->attn_factor : (float)(0.1 * log(sc->factor) + 1.0);
    }
    for (int i = 0; i < n_rot / 2; i++) {
        const double f = 1.0 / pow((double)theta, (double)(2 * i) / n_rot);
        double keep = 1.0; /* how much of f stays, the rest divided by factor */
        if (kind == SDY_ROPE_LINEAR) keep = 0.0;
        if (kind == SDY_ROPE_YARN) keep = 1.0 - fmin(fmax((i - low) / fmax(high - low, 1e-3), 0.0), 1.0);
        if (kind == SDY_ROPE_LLAMA3)
            keep = fmin(fmax((sc->orig_ctx * f / TWO_PI - sc->low_freq) / ((double)sc->high_freq - sc->low_freq), 0.0), 1.0);
        freq[i] = keep == 1.0 ? f : f * keep + f / sc->factor * (1.0 - keep);
    }
    return 0;
}
