"""Plain 64-bit forms of the operators that verify drafted tokens, for their
tests: the oracle's scalar functions row by row, Python integers and numpy for
what the oracle has no counterpart of (scaled frequencies, masks, penalties)."""
from __future__ import annotations

import ctypes as C

import numpy as np

import oracle_lib

ONE = 1 << 32
TWO_PI = 26986075409
I32_MIN, I32_MAX = -(2**31), 2**31 - 1


def half_even(n: int, d: int) -> int:
    """n / d to the nearest integer, ties to even (Python integers, d > 0)."""
    q, r = divmod(n, d)
    return q + (2 * r > d or (2 * r == d and q & 1))


def sat(v: int) -> int:
    return max(I32_MIN, min(I32_MAX, v))


def mul_sat(a: int, b: int) -> int:
    return sat(half_even(a * b, 65536))


def frequencies(base: int, freq_base_dim: int, pairs: int, scaling: int = 0, factor: int = ONE, low: int = 0,
                high: int = 0, original: int = 0) -> list[int]:
    freq = [int(f) for f in oracle_lib.rope_inv_frequencies(base, freq_base_dim, pairs)] if pairs else []
    out = []
    for f in freq:
        g = half_even(f << 32, factor)
        if scaling == 0:
            out.append(f)
        elif scaling == 1:
            out.append(g)
        else:
            turns = half_even(original * f << 32, TWO_PI)
            w = ONE if turns >= high else 0 if turns <= low else half_even((turns - low) << 32, high - low)
            out.append(half_even(w * f, ONE) + half_even((ONE - w) * g, ONE))
    return out


def head_row(x: np.ndarray, gain, eps: int, norm: bool, freq, position: int, layout: int, amplitude: int,
             rotate: bool) -> np.ndarray:
    """One head row: the oracle's norms, then the pairs turned one by one."""
    L = oracle_lib.lib()
    x = np.ascontiguousarray(x, dtype=np.int32).copy()
    if norm:
        if gain is None:
            oracle_lib.check(L.orc_value_rms_norm(oracle_lib.ptr(x), x.size, eps), True)
        else:
            g = np.ascontiguousarray(gain, dtype=np.int32)
            oracle_lib.check(L.orc_rms_norm(oracle_lib.ptr(x), oracle_lib.ptr(g), x.size, eps), True)
    if rotate:
        pairs = len(freq)
        for i, f in enumerate(freq):
            c, s = C.c_int32(), C.c_int32()
            L.orc_sin_cos_acc(min(position * f, 2**63 - 1), C.byref(c), C.byref(s))
            cv, sv = mul_sat(c.value, amplitude), mul_sat(s.value, amplitude)
            ia, ib = (i, i + pairs) if layout == 0 else (2 * i, 2 * i + 1)
            a, b = int(x[ia]), int(x[ib])
            x[ia] = sat(mul_sat(a, cv) - mul_sat(b, sv))
            x[ib] = sat(mul_sat(b, cv) + mul_sat(a, sv))
    return x


def attention_row(q: np.ndarray, keys: np.ndarray, values: np.ndarray) -> np.ndarray:
    """One (row, head) over its visible keys and values [n][head_dim]."""
    L = oracle_lib.lib()
    hd, n = q.size, len(keys)
    out = np.zeros(hd, dtype=np.int32)
    if n == 0:
        return out
    q, keys, values = (np.ascontiguousarray(t, dtype=np.int32) for t in (q, keys, values))
    score, w = np.empty(n, dtype=np.int32), np.empty(n, dtype=np.int32)
    one = C.c_int32()
    for r in range(n):
        oracle_lib.check(L.orc_attention_score(oracle_lib.ptr(q), oracle_lib.ptr(keys[r]), hd, C.byref(one)), True)
        score[r] = one.value
    oracle_lib.check(L.orc_attention_softmax(oracle_lib.ptr(score), n, oracle_lib.ptr(w)), True)
    oracle_lib.check(L.orc_attention_weighted_sum(oracle_lib.ptr(w), oracle_lib.ptr(values), n, hd, oracle_lib.ptr(out)),
                     True)
    return out


def attention_tree(caches, drafts, q, k, v, masks, starts, heads: int, kv_heads: int, hd: int) -> np.ndarray:
    """caches: per sequence (k rows, v rows) in logical order [n][kv_heads * hd]."""
    out, at = np.zeros((sum(drafts), heads * hd), dtype=np.int32), 0
    for (ck, cv), d in zip(caches, drafts):
        for i in range(d):
            n = len(ck)
            start = min(int(starts[at + i]) if starts is not None else 0, n)
            seen = [j for j in range(d) if int(masks[at + i]) >> j & 1]
            for h in range(heads):
                c = slice((h // (heads // kv_heads)) * hd, (h // (heads // kv_heads) + 1) * hd)
                kk = np.concatenate([ck[start:, c], k[at:at + d, c][seen]])
                vv = np.concatenate([cv[start:, c], v[at:at + d, c][seen]])
                out[at + i, h * hd:(h + 1) * hd] = attention_row(q[at + i, h * hd:(h + 1) * hd], kk, vv)
        at += d
    return out


def bits(w, scale=None) -> np.ndarray:
    """Weight bits of an int8 x row scale or i16 / i32 matrix."""
    w = np.asarray(w).astype(np.int64)
    return (w if scale is None else w * np.asarray(scale, dtype=np.int64)[:, None]).astype(np.int32)


def linear_adapters(w: np.ndarray, adapters, x: np.ndarray, index) -> np.ndarray:
    """w: weight bits; adapters: (down bits, up bits, scale)."""
    out = np.empty((len(x), w.shape[0]), dtype=np.int32)
    for t, row in enumerate(x):
        y = oracle_lib.det_linear(w, row).astype(np.int64)
        if int(index[t]) < len(adapters):
            down, up, scale = adapters[int(index[t])]
            d = oracle_lib.det_linear(up, oracle_lib.det_linear(down, row)).astype(object)
            y = np.array([sat(int(a) + mul_sat(int(b), scale)) for a, b in zip(y, d)], dtype=np.int64)
        out[t] = y
    return out


def select(logits: np.ndarray, penalties=None, ids=None, spans=None, bias=None, mask=None):
    """logits [n][vocab]; spans: per row a list of (begin, end); bias: per row a list of (token, value)."""
    n, vocab = logits.shape
    out, tokens = np.empty_like(logits), np.full(n, 0xFFFFFFFF, dtype=np.uint32)
    for r in range(n):
        x = [int(v) for v in logits[r]]
        add = [0] * vocab
        if penalties is not None and spans is not None:
            count = {}
            for b, e in spans[r]:
                for t in ids[b:min(e, len(ids))]:
                    if t < vocab:
                        count[int(t)] = count.get(int(t), 0) + 1
            rep, freq, pres = (int(p) for p in penalties[r])
            for t, c in count.items():
                if rep > 0:
                    x[t] = sat(half_even(x[t] * 65536, rep)) if x[t] > 0 else mul_sat(x[t], rep)
                add[t] -= c * freq + pres
        for t, b in (bias[r] if bias is not None else []):
            if t < vocab:
                add[t] += int(b)
        x = [sat(a + b) for a, b in zip(x, add)]
        ok = range(vocab) if mask is None else [t for t in range(vocab) if int(mask[r][t // 32]) >> (t % 32) & 1]
        if mask is not None:
            allowed = set(ok)
            x = [v if t in allowed else I32_MIN for t, v in enumerate(x)]
        out[r] = x
        best = max((x[t] for t in ok), default=None)
        if best is not None:
            tokens[r] = next(t for t in ok if x[t] == best)
    return out, tokens
