/*
 * neurosim_hip_signal.h -- C ABI of the signal operators around the tick: the short
 * causal convolution per channel, the selective state space scan and the gated linear
 * recurrence, each for whole signals, for one tick, and backwards.  Conventions (status codes, ns_last_error,
 * caller's stream, no allocation, no synchronisation) are those of neurosim_hip.h.
 *
 * A signal is [T, B, N]: ticks, columns, channels, element (t, b, n) at
 * data[t*stride_t + b*stride_b + n].  All signals of a call share one element type.
 * `lengths` (optional, device int32[B]) gives each column's own number of ticks,
 * clamped to [0, T]: later ticks of that column give zeros and change nothing, and
 * what their inputs hold is never used.  What a call writes overlaps nothing that it
 * reads, but for the history or state that a step moves on in place.
 */
#ifndef NEUROSIM_HIP_SIGNAL_H
#define NEUROSIM_HIP_SIGNAL_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
#define NS_TYPE_F32 0
#define NS_TYPE_BF16 1
#define NS_TYPE_F16 2

/* Strides in elements; data NULL: absent. */
typedef struct ns_signal {
  void* data;
  int64_t stride_t;
  int64_t stride_b;
} ns_signal;

/* Largest number of taps and of states per channel. */
#define NS_CONV_MAX_TAPS 8
#define NS_SCAN_MAX_STATES 64

/* Causal convolution per channel, W taps:
 *   p[t,b,n] = bias[n] + sum_k weight[n,k] * x[t-W+1+k, b, n],   y = p or silu(p)
 * with x at tick -1, -2, ... taken from `history` (rows W-2, W-3, ...; absent: 0). */
typedef struct ns_conv_args {
  int64_t ticks, batch, channels;
  int32_t taps;                /* W, 1 .. NS_CONV_MAX_TAPS */
  int32_t type;                /* NS_TYPE_* of x, y, history (float32 sums) */
  int32_t silu;                /* nonzero: y = silu(p) */
  int32_t chunk;               /* ticks per thread; 0: chosen by ns_conv_chunk */
  ns_signal x;
  const float* weight;         /* [N][W] */
  const float* bias;           /* [N] or NULL */
  ns_signal history;           /* [W-1, B, N] before the first tick, or absent */
  const int32_t* lengths;
  ns_signal y;
  ns_signal out_history;       /* [W-1, B, N]: the last W-1 inputs; absent: not written.
                                  May be `history` itself in ns_conv_step only */
  /* ns_conv_backward only: */
  ns_signal dy;                /* gradient of y */
  ns_signal dout_history;      /* gradient of out_history, or absent */
  ns_signal dx;                /* absent: not written */
  ns_signal dhistory;          /* absent: not written */
  float* partials;             /* workspace (ns_conv_backward_floats) */
  float* dweight;              /* [N][W], and the bias gradient [N] behind it */
} ns_conv_args;

/* Ticks per thread that ns_conv_forward (`backward` zero) and ns_conv_backward use. */
int64_t ns_conv_chunk(int64_t ticks, int64_t batch, int64_t channels, int32_t type,
                      int32_t backward);
/* Floats of ns_conv_backward's workspace (with `chunk` 0). */
int64_t ns_conv_backward_floats(int64_t ticks, int64_t batch, int64_t channels, int32_t taps,
                                int32_t type);
int ns_conv_forward(const ns_conv_args* args, void* stream);
/* One tick (ticks == 1, no lengths), `out_history` the history itself, moved on in place. */
int ns_conv_step(const ns_conv_args* args, void* stream);
/* Gradients, with sums in a fixed order (no atomics). */
int ns_conv_backward(const ns_conv_args* args, void* stream);

/* Selective scan, S states per channel, channels in G groups of N/G neighbours that
 * share B and C (group of channel n: n / (N/G)):
 *   dt = softplus(delta + delta_bias)           (or delta + delta_bias)
 *   h[t,b,n,s] = exp(dt A[n,s]) h[t-1] + dt x B[t,b,g,s]
 *   y[t,b,n]   = (sum_s C[t,b,g,s] h[t] + D[n] x) silu(z)     (D, z: optional) */
typedef struct ns_scan_args {
  int64_t ticks, batch, channels, groups;
  int32_t states;              /* S, 1 .. NS_SCAN_MAX_STATES */
  int32_t type;                /* NS_TYPE_* of x, delta, z, B, C, y (states, A, D float32) */
  int32_t softplus;
  int32_t chunks;              /* time chunks scanned side by side (ns_scan_plan) */
  ns_signal x, delta, z, y;    /* z optional */
  ns_signal write, read;       /* B and C: [T, B, G, S], (g, s) at g*S + s of a column */
  const float* rates;          /* A [N][S] */
  const float* skip;           /* D [N] or NULL */
  const float* delta_bias;     /* [N] or NULL */
  const float* state;          /* h before the first tick [B][N][S], or NULL: zeros */
  float* out_state;            /* h after each column's last tick [B][N][S] */
  const int32_t* lengths;
  float* checkpoints;          /* optional workspace (ns_scan_plan): h before every tile of
                                  ticks, kept for ns_scan_backward */
  float* ends;                 /* workspace (ns_scan_plan; chunks > 1) */
  /* ns_scan_backward only (checkpoints required): */
  ns_signal dy;
  const float* dout_state;     /* gradient of out_state, or NULL: zeros */
  ns_signal dx, ddelta, dz;    /* dz present exactly if z is */
  ns_signal dwrite, dread;     /* dB, dC */
  float* dstate;               /* gradient of state [B][N][S], or NULL */
  float* dparameters;          /* dA [N][S], then dD [N] and d(delta_bias) [N] (these are
                                  written also without D and without a bias) */
  float* partials;             /* workspace (ns_scan_plan) */
} ns_scan_args;

/* What a scan of this shape needs: sizes[0] time chunks worth scanning side by side (1: none),
 * the same in both directions, and with that many chunks the floats of `ends` [1] (0 for one
 * chunk), of `checkpoints` [2], and of the `backward`'s `partials` [3] (0 for a forward). */
int ns_scan_plan(int64_t ticks, int64_t batch, int64_t channels, int64_t groups, int32_t states,
                 int32_t backward, int64_t* sizes);
int ns_scan_forward(const ns_scan_args* args, void* stream);
/* One tick (ticks == 1, no lengths): `out_state` is the state itself, updated in place. */
int ns_scan_step(const ns_scan_args* args, void* stream);
int ns_scan_backward(const ns_scan_args* args, void* stream);

/* Gated linear recurrence, one state per channel:
 *   s = sigmoid(forget), i = sigmoid(write), a = exp(-rates[n] s)
 *   h[t,b,n] = a h[t-1] + sqrt(1 - a^2) i x,   y = h silu(z)   (z optional)
 * Rates are not negative (a negative one counts as 0, and its gradient is 0). */
typedef struct ns_recurrence_args {
  int64_t ticks, batch, channels;
  int32_t type;                /* NS_TYPE_* of all signals (states and rates float32) */
  int32_t chunks;              /* time chunks walked side by side (ns_recurrence_plan) */
  ns_signal x, forget, write, z, y;
  const float* rates;          /* [N] */
  const float* state;          /* h before the first tick [B][N], or NULL: zeros */
  float* out_state;            /* h after each column's last tick [B][N], or NULL */
  const int32_t* lengths;
  float* checkpoints;          /* optional workspace (ns_recurrence_plan): states kept for
                                  ns_recurrence_backward */
  float* ends;                 /* workspace (ns_recurrence_plan; chunks > 1) */
  /* ns_recurrence_backward only (checkpoints required): */
  ns_signal dy;
  const float* dout_state;     /* gradient of out_state, or NULL: zeros */
  ns_signal dx, dforget, dwrite, dz;   /* dz present exactly if z is */
  float* dstate;               /* gradient of state [B][N], or NULL */
  float* drates;               /* [N] */
  float* partials;             /* workspace (ns_recurrence_plan) */
} ns_recurrence_args;

/* What a recurrence of this shape needs: sizes[0] time chunks worth walking side by side (1:
 * none), and with that many the floats of `ends` [1] (0 for one chunk), of `checkpoints` [2] and of
 * ns_recurrence_backward's `partials` [3]. */
int ns_recurrence_plan(int64_t ticks, int64_t batch, int64_t channels, int32_t type,
                       int64_t* sizes);
int ns_recurrence_forward(const ns_recurrence_args* args, void* stream);
/* One tick (ticks == 1, no lengths): `out_state` is the state itself, updated in place. */
int ns_recurrence_step(const ns_recurrence_args* args, void* stream);
/* Gradients, with sums in a fixed order (no atomics). */
int ns_recurrence_backward(const ns_recurrence_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif  /* NEUROSIM_HIP_SIGNAL_H */
