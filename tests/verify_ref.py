"""Verification of drafted tokens in 64 bits on the CPU, sequence by sequence
from the definition in include/spock_hip.h."""
import math

import numpy as np


def _dist(row, kind, temp):
    if kind == "probs":
        return row.astype(np.float64)
    with np.errstate(all="ignore"):
        x = row.astype(np.float64)
        e = np.exp((x - x.max()) / temp)
        return e / e.sum()


def _argmax(row):
    """Lowest index of the largest value above -inf, NaN aside; -1 where there is none."""
    x = np.where(np.isnan(row), -np.inf, row.astype(np.float64))
    i = int(np.argmax(x))
    return i if x[i] > -np.inf else -1


def verify(target, tokens, cu, u_accept, u_sample, draft=None, kind="logits", temperature=None, context=None):
    """(out_tokens, accepted, logprobs, context_out); rows of no sequence keep -99 and NaN."""
    T, V = target.shape
    S = len(u_sample)
    out, logp = np.full(T, -99, np.int64), np.full(T, math.nan)
    accepted = np.zeros(S, np.int64)
    for s in range(S):
        a = min(max(int(cu[s]), 0), T)
        b = max(a, min(int(cu[s + 1]), T))
        temp = 1.0 if temperature is None else float(temperature[s])
        greedy = not temp > 0
        temp = 1.0 if greedy else temp
        for t in range(a, b):
            out[t], logp[t] = -1, 0.0
        for t in range(a, b):
            p = _dist(target[t], kind, temp)
            d = int(tokens[t + 1]) if t + 1 < b else None
            token = None
            if d is not None and 0 <= d < V:
                q = None if draft is None else _dist(draft[t], kind, temp)
                if greedy:
                    yes = _argmax(target[t]) == d
                else:
                    yes = float(u_accept[t]) * (1.0 if q is None else q[d]) < p[d]
                if yes:
                    token = d
                    accepted[s] += 1
            if token is None:
                if greedy:
                    token = _argmax(target[t])
                else:
                    w = p
                    if d is not None:
                        if draft is None:
                            w = p.copy()
                            if 0 <= d < V:
                                w[d] = 0.0
                        else:
                            w = p - _dist(draft[t], kind, temp)
                            w = np.where(w < 0, 0.0, w)
                    if not w.sum() > 0:
                        w = p
                    c = np.cumsum(w)
                    token = -1
                    if c[-1] > 0:
                        past = np.nonzero(c > float(u_sample[s]) * c[-1])[0]
                        token = int(past[0]) if past.size else int(np.nonzero(w > 0)[0][-1])
                stop = True
            else:
                stop = False
            out[t] = token
            if token >= 0:
                with np.errstate(all="ignore"):
                    x = target[t].astype(np.float64)
                    if kind == "probs":
                        logp[t] = np.log(x[token])
                    else:
                        m = x.max()
                        logp[t] = (x[token] - m) / temp - np.log(np.exp((x - m) / temp).sum())
            if stop:
                break
    ctx = None
    if context is not None:
        n = [max(0, min(max(int(cu[s + 1]), min(max(int(cu[s]), 0), T)), T) - min(max(int(cu[s]), 0), T)) for s in range(S)]
        ctx = np.array([int(context[s]) - max(0, n[s] - 1 - accepted[s]) for s in range(S)])
    return out, accepted, logp, ctx
