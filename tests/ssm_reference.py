"""The mixer's recurrence in 64 bits, token by token, with bounds on what
single precision may differ by.

bound(): every product and sum of an fp32 evaluation rounds by at most u =
2^-24 of its value, and what it rounds is at most the same expression over
absolute values.  An output's longest chain is: the convolution and silu of
x, B and C (conv_width + 8 roundings each), dt (its relative error of about 8 u
moves a decay e^-c by 8 u c e^-c < 3 u), the sum over the state (N, or N / 2
with fewer), the sum over a chunk of 32 tokens, one product with a decay per
chunk and segment, and the skip.  K roundings move it by at most K u of the
absolute expression (to first order, K u < 1e-3 here).

Near the end of single precision's range a product of the state is off by more
than u of itself: its operands are at best 2^100 x 2^14 times x dt B / |B|, whose
f16 parts are multiples of 2^-24, so off by 2^-25, and 2^14 B / |B|, below 2^15.
The product is off by 2^(-25 + 15 - 114) = 2^-124 (the smallest normal number is
2^-126): each token adds that to its state.
"""
import numpy as np

U = 2.0 ** -24


def _silu(v):
    return v / (1 + np.exp(-v))


def _softplus(v):
    return np.maximum(v, 0) + np.log1p(np.exp(-np.abs(v)))


def sequence(layer, x, conv, ssm):
    """One sequence: (y, conv, ssm, y's bound, ssm's bound) for rows x [T][row] from a state."""
    L, H, P, G, N, W = layer, layer.heads, layer.head_dim, layer.groups, layer.state, layer.conv_width
    x = x.astype(np.float64)
    T, inner, channels = x.shape[0], L.inner, L.channels
    raw = np.concatenate([conv.astype(np.float64), x[:, inner:inner + channels]])
    bias = np.zeros(channels) if L.conv_bias is None else L.conv_bias.astype(np.float64)
    w = L.conv_weight.astype(np.float64)
    s = ssm.astype(np.float64)
    s_abs = np.abs(s)
    K = 3 * (W + 8) + N + 32 + T // 16 + 32
    lost = 2.0 ** -124 / (K * U)
    y, y_abs = np.empty((T, inner)), np.empty((T, inner))
    share = H // G
    a, d = L.a.astype(np.float64), L.d.astype(np.float64)
    for t in range(T):
        taps = raw[t:t + W]
        pre = bias + (w.T * taps).sum(0)
        # |silu'| <= 1.1, so the convolution's roundings reach u by the taps' absolute sum
        u, u_abs = _silu(pre), np.abs(bias) + (np.abs(w.T) * np.abs(taps)).sum(0)
        dt = _softplus(x[t, inner + channels:] + L.dt_bias.astype(np.float64))
        e = np.exp(dt * a)
        xs = u[:inner].reshape(H, P)
        bs = np.repeat(u[inner:inner + G * N].reshape(G, N), share, 0)
        cs = np.repeat(u[inner + G * N:].reshape(G, N), share, 0)
        xa = u_abs[:inner].reshape(H, P)
        ba = np.repeat(u_abs[inner:inner + G * N].reshape(G, N), share, 0)
        ca = np.repeat(u_abs[inner + G * N:].reshape(G, N), share, 0)
        s = e[:, None, None] * s + (dt[:, None] * xs)[:, :, None] * bs[:, None, :]
        s_abs = e[:, None, None] * s_abs + (dt[:, None] * xa)[:, :, None] * ba[:, None, :] + lost
        y[t] = ((s * cs[:, None, :]).sum(-1) + d[:, None] * xs).reshape(-1)
        y_abs[t] = ((s_abs * ca[:, None, :]).sum(-1) + np.abs(d)[:, None] * xa).reshape(-1)
    z = _silu(x[:, :inner])
    v, dv = y * z, K * U * y_abs * np.abs(z) + 8 * U * np.abs(y * z)
    vg, dg = v.reshape(T, G, inner // G), dv.reshape(T, G, inner // G)
    r = 1 / np.sqrt((vg * vg).mean(-1, keepdims=True) + float(np.float32(L.norm_epsilon)))
    norm = L.norm.astype(np.float64)
    out = (vg * r).reshape(T, inner) * norm
    # d(1 / rms) / (1 / rms) <= |dv| / |v| in the 2-norm over the group, and its own roundings
    rel = np.sqrt((dg * dg).sum(-1, keepdims=True)) * r / np.sqrt(vg.shape[-1]) + 24 * U
    bound = (r * (dg + np.abs(vg) * rel)).reshape(T, inner) * np.abs(norm)
    return out, raw[T:].astype(np.float32), s, bound, K * U * s_abs


# What all outputs of a call, or all elements of its states, may differ by together: the 2-norm of the error over
# the 2-norm of the result, for ordinary inputs.  The bounds above are for the worst case, every rounding of the
# longest chain one way and every term of a sum in line, and a product of half the digits would stay within them.
# Together, roundings are of either sign: one is off by 0.4 U of its value in the mean of squares, and about 45 of
# them follow one another on a full value (the convolution and silu of x, B and C, the step and its decay, a product,
# a sum in a tree, the skip, the gate and the norm), so 0.4 U sqrt(45) = 2.7 U = 1.6e-7; three times that is allowed.
TOGETHER = 8 * U


def with_operands(layer, x, conv, ssm, operand):
    """(y, ssm) of a sequence whose products take operand(name, v) of x dt ("x"), B, C and the state ("s")."""
    H, P, G, N, W, inner = layer.heads, layer.head_dim, layer.groups, layer.state, layer.conv_width, layer.inner
    x, s = x.astype(np.float64), ssm.astype(np.float64)
    T, channels = len(x), layer.channels
    raw = np.concatenate([conv, x[:, inner:inner + channels]])
    u = np.zeros(channels) if layer.conv_bias is None else layer.conv_bias
    u = _silu(u + sum(layer.conv_weight[:, k].astype(np.float64) * raw[k:k + T] for k in range(W)))
    dt = _softplus(x[:, inner + channels:] + layer.dt_bias)
    heads = u[:, :inner].reshape(T, H, P)
    b, c = (np.repeat(v.reshape(T, G, N), H // G, 1) for v in (u[:, inner:inner + G * N], u[:, inner + G * N:]))
    left, b, c = operand("x", dt[:, :, None] * heads), operand("B", b), operand("C", c)
    y = np.empty((T, H, P))
    for t in range(T):
        s = np.exp(dt[t] * layer.a)[:, None, None] * s + left[t][:, :, None] * b[t][:, None, :]
        y[t] = (operand("s", s) * c[t][:, None, :]).sum(-1) + layer.d[:, None] * heads[t]
    v = (y.reshape(T, inner) * _silu(x[:, :inner])).reshape(T, G, -1)
    v = v / np.sqrt((v * v).mean(-1, keepdims=True) + layer.norm_epsilon)
    return v.reshape(T, inner) * layer.norm, s


def together(got, want):
    return float(np.sqrt(((got - want) ** 2).sum() / (want ** 2).sum()))
