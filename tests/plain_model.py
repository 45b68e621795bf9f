"""A Qwen2 forward pass in 64 bits whose K and V rows go through a cache's type, for the
tests of models over a quantised cache."""
import ctypes as C

import numpy as np

import kv_plain


def _vec(ptr, n):
    return np.ctypeslib.as_array((C.c_float * n).from_address(ptr)).astype(np.float64) if ptr else np.zeros(n)


class PlainModel:
    def __init__(self, lrs, orc, sm, cfg):
        self.lrs, self.cfg = lrs, cfg
        self.hd, self.nh, self.nkv = cfg.resolved_head_dim(), cfg.num_attention_heads, cfg.num_key_value_heads
        h, d = cfg.hidden_size, sm.desc().contents

        def mat(name, layer=None):
            t = sm.tensor(name, layer)
            return orc.dequantize(t.data, int(t.quant_type), t.rows(), t.cols()).astype(np.float64)
        self.embed, self.head, self.norm = mat("embed"), mat("lm_head"), _vec(d.final_norm, h)
        self.layers = []
        for i in range(cfg.num_hidden_layers):
            f = d.layers[i]
            w = {n[0]: mat(n, i) for n in ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj")}
            kvw = self.nkv * self.hd
            w.update(in_norm=_vec(f.input_layernorm, h), post_norm=_vec(f.post_attention_layernorm, h),
                     qb=_vec(f.q_bias, h), kb=_vec(f.k_bias, kvw), vb=_vec(f.v_bias, kvw))
            self.layers.append(w)

    def rotate(self, x, pos):
        half = self.hd // 2
        f32 = np.float32
        freq = f32(1) / np.power(f32(self.cfg.rope_theta), f32(2) * np.arange(half, dtype=f32) / f32(self.hd))
        angle = (np.asarray(pos, f32)[:, None] * freq[None]).astype(np.float64)[:, None, :]
        a, b = x[..., :half], x[..., half:]
        return np.concatenate([a * np.cos(angle) - b * np.sin(angle), a * np.sin(angle) + b * np.cos(angle)], -1)

    def logits(self, tokens, kv, split=None):
        """[n, vocab]: the logits after each token, every K and V row held as `kv` holds it;
        `split` restates what a kernel's dot products make of a row of x."""
        n, eps, hold = len(tokens), self.cfg.rms_norm_eps, lambda x: kv_plain.held(self.lrs, kv, x.astype(np.float32))

        def dot(x, w):
            return (x if split is None else np.array([split(r.astype(np.float32)) for r in x])) @ w.T

        def norm(x, w):
            return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
        x = self.embed[np.asarray(tokens)]
        pos, seen = np.arange(n), np.tril(np.ones((n, n), bool))
        for w in self.layers:
            y = norm(x, w["in_norm"])
            q = self.rotate((dot(y, w["q"]) + w["qb"]).reshape(n, self.nh, self.hd), pos)
            k = hold(self.rotate((dot(y, w["k"]) + w["kb"]).reshape(n, self.nkv, self.hd), pos))
            v = hold((dot(y, w["v"]) + w["vb"]).reshape(n, self.nkv, self.hd))
            att = np.empty((n, self.nh, self.hd))
            for h in range(self.nh):
                s = q[:, h] @ k[:, h * self.nkv // self.nh].T / np.sqrt(self.hd)
                p = np.where(seen, np.exp(np.where(seen, s - np.where(seen, s, -np.inf).max(1, keepdims=True), 0.0)), 0.0)
                att[:, h] = p / p.sum(1, keepdims=True) @ v[:, h * self.nkv // self.nh]
            x = x + dot(att.reshape(n, -1), w["o"])
            y = norm(x, w["post_norm"])
            g = dot(y, w["g"])
            x = x + dot(g / (1.0 + np.exp(-g)) * dot(y, w["u"]), w["d"])
        return dot(norm(x, self.norm), self.head)
