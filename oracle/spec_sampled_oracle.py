"""The rejection rule of hi_rocm_spec_verify_sampled in 64 bits on the CPU.
Test infrastructure only."""
import numpy as np


def _draw(r, u):
    r = np.where(r > 0, r, 0.0)  # (NaN: 0)
    mass = np.cumsum(r)
    if not mass[-1] > 0:
        return None
    over = np.nonzero((mass > u * mass[-1]) & (r > 0))[0]
    return int(over[0]) if len(over) else int(np.nonzero(r > 0)[0][-1])


def verify(target, tokens, uniforms, draft=None, lengths=None):
    """target [batch][K + 1][V], draft [batch][K][V] (float64 arrays), tokens
    [batch][K], uniforms [batch][K + 1] -> tokens int32 [batch][K + 1] (-1 behind
    the drawn one), counts int32 [batch]."""
    B, K, V = target.shape[0], target.shape[1] - 1, target.shape[2]
    out, counts = np.full((B, K + 1), -1, np.int32), np.zeros(B, np.int32)
    for b in range(B):
        k = K if lengths is None else min(max(int(lengths[b]), 0), K)
        n = 0
        while n < k:
            t, u = int(tokens[b, n]), float(uniforms[b, n])
            if not 0 <= t < V:
                break
            q = 1.0 if draft is None else draft[b, n, t]
            if not u * q < target[b, n, t]:
                break
            out[b, n] = t
            n += 1
        p, u = target[b, n], float(uniforms[b, K])
        token = None
        if n < k:
            q = np.zeros(V) if draft is None else draft[b, n]
            if draft is None and 0 <= int(tokens[b, n]) < V:
                q[int(tokens[b, n])] = 1.0
            token = _draw(p - q, u)
        if token is None:
            token = _draw(p, u)
        out[b, n] = 0 if token is None else token
        counts[b] = n + 1
    return out, counts
