"""Whole models on 4-bit caches (hip_lm_batch_new_kv4) in numpy: fp32 products and
experts by the oracle, the caches and the attention in 64 bits (kv_ref.py)."""
import numpy as np

import hipkv
import kv_ref
import oracle

HL = 128


def norm(x, w):
    x = np.asarray(x, np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5) * w


class Sequence:
    """One sequence's forward: logits of chosen rows, and how close its routing
    came to another choice."""

    def __init__(self, md, ids, bits4=True, rows=None):
        E, H, L, wt, K = md["E"], md["H"], md["layers"], md["wtype"], md["K"]
        KH, window = md.get("KH", H), md.get("window", 0)
        olmoe = md["arch"] == "olmoe"
        T = len(ids)
        rows = np.arange(T) if rows is None else np.asarray(rows)
        freq = md["theta"] ** (-2.0 * np.arange(HL // 2) / HL)
        self.gap = np.ones(T)
        table = np.asarray(md["token_embd"]).reshape(md["V"], -1)
        h = np.stack([oracle.dequant(table[i], wt, E) for i in ids]).astype(np.float64)
        for l, b in enumerate(md["blk"]):
            x = norm(h, b["attn_norm"])
            q, k, v = (oracle.qmat_mul(x, b[n], wt, N, E).astype(np.float64)
                       for n, N in (("q", H * HL), ("k", KH * HL), ("v", KH * HL)))
            if olmoe:
                q, k = norm(q, b["q_norm"]), norm(k, b["k_norm"])
            q = kv_ref.rotate(q.reshape(T, H, HL), np.arange(T), freq, 1.0, hipkv.PAIRS)
            k = kv_ref.rotate(k.reshape(T, KH, HL), np.arange(T), freq, 1.0, hipkv.PAIRS)
            v = v.reshape(T, KH, HL)
            if bits4:
                c, d = kv_ref.quantize(k.reshape(T, KH, HL // 32, 32))
                k = ((c - 8.0) * d[..., None].astype(np.float64)).reshape(T, KH, HL)
                c, d = kv_ref.quantize(v)
                v = (c - 8.0) * d[..., None].astype(np.float64)
            at = rows if l == L - 1 else np.arange(T)
            o = np.zeros((len(at), H, HL))
            for n, p in enumerate(at):
                o[n] = kv_ref.attend(q[p], k[:p + 1], v[:p + 1], int(p), HL ** -0.5, window)[0]
            h = h[at] + oracle.qmat_mul(o.reshape(len(at), -1), b["o"], wt, E, H * HL)
            lay = dict(router=b["router"], gate=b["gate"], up=b["up"], down=b["down"], wtype=wt,
                       E=E, EI=md["EI"], NE=md["NE"])
            y, _, _, _, pr = oracle.moe_ffn(norm(h, b["ffn_norm"]), lay, K, not olmoe)
            if K < md["NE"]:
                s = np.sort(pr, axis=1)[:, ::-1]
                self.gap[at] = np.minimum(self.gap[at], (s[:, K - 1] - s[:, K]) / s[:, K - 1])
            h = h + y
        self.logits = oracle.qmat_mul(norm(h, md["output_norm"]), md["output"], wt, md["V"],
                                      E).astype(np.float64)
