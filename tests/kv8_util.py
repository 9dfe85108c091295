"""Attention over caches of 8 bits, restated in f64 numpy: random projections in the library's layout, what a cache has to hold for them, and the attention's output over the values that a
cache holds (include/bitnet_hip.h section 5, kv8_*)."""
import numpy as np

from oracle import stack_oracle as so
from tests import stack_util as u

f64 = np.float64


def numbers_of(x):
    """f32 vectors along the last axis -> (numbers, scales) by the rule, every operation rounded to f32"""
    x = np.asarray(x, np.float32)
    a = np.abs(x).max(-1)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        live, finite = a >= np.float32(1.5e-36), np.isfinite(x).all(-1)
        scale = np.where(finite, np.where(live, a / np.float32(127), np.float32(0)), np.float32("nan")).astype(np.float32)
        factor = np.where(live & finite, np.float32(127) / a, np.float32(0)).astype(np.float32)
        n = np.where(finite[..., None], np.rint(x * factor[..., None]), 0)
    return n.astype(np.int8), scale


def unpack(cache):
    """values int8 [kv][capacity / 32][vdimp / 32][16][4][2][8] -> [kv][capacity][vdimp]"""
    g, t, c = cache.shape[:3]
    return cache.transpose(0, 1, 4, 6, 2, 5, 3).reshape(g, t * 32, c * 32)


def pack(values):
    g, p, v = values.shape
    return np.ascontiguousarray(values.reshape(g, p // 32, 4, 8, v // 32, 2, 16).transpose(0, 1, 4, 6, 2, 5, 3))


class Cache:
    """device buffers of one cache; `fill`: what lies there before anything is written"""

    def __init__(self, kv, maps, capacity, dimp, vdimp, fill=0, scale=0.0):
        import torch

        self.k = torch.full((kv, maps, capacity, dimp), fill, dtype=torch.int8, device="cuda")
        self.v = torch.full((kv, capacity // 32, vdimp // 32, 16, 4, 2, 8), fill, dtype=torch.int8, device="cuda")
        self.ks, self.vs = torch.full((kv, maps, capacity), scale, device="cuda"), torch.full((kv, capacity), scale, device="cuda")

    def host(self):
        """numbers and scales: keys, values [kv][capacity][vdimp]"""
        return self.k.cpu().numpy(), unpack(self.v.cpu().numpy()), self.ks.cpu().numpy(), self.vs.cpu().numpy()

    def held(self):
        k, v, ks, vs = self.host()
        return k.astype(f64) * ks[..., None].astype(f64), v.astype(f64) * vs[..., None].astype(f64)


class Attention:
    """n tokens' projections and everything that stands ahead of the attention"""

    def __init__(self, pkg, n, heads, kv, dim, vdim, maps=1, normed=True, rot=0, window=0, chunk=0, sink=False, gate=None, far=False, taps=0, keys_as_values=False, f32=False, sharp=1.0,
                 fill=0, scale=0.0, seed=0, capacity=None):
        g = np.random.default_rng([n, heads, dim, vdim, maps, window, chunk, taps, seed])
        self.pkg, self.n, self.heads, self.kv, self.maps, self.dim, self.vdim, self.f32, self.taps, self.rot = pkg, n, heads, kv, maps, dim, vdim, f32, taps, rot
        self.window, self.chunk, self.gate = window, chunk, gate
        self.dimp, self.vdimp, self.cap = u.up_to(dim, 32), u.up_to(vdim, 32), capacity or u.up_to(n, 128)
        store = (lambda a: a.astype(np.float32)) if f32 else u.rounded
        raw = [store(g.standard_normal((n, heads * maps, dim)) * 1.4), store(g.standard_normal((n, kv * maps, dim)) * np.exp(0.4 * g.standard_normal(dim)))]
        raw.append(raw[1] if keys_as_values else store(g.standard_normal((n, kv, vdim)) * np.exp(0.4 * g.standard_normal((n, kv, 1)))))
        parts = [u.padded(a, to).reshape(n, -1) for a, to in zip(raw[:2] if keys_as_values else raw, (self.dimp, self.dimp, self.vdimp))]
        self.channels = sum(a.shape[1] for a in parts)
        self.z = store(2.0 * g.standard_normal((n, heads * (self.vdimp if gate == "columns" else 1))))
        self.rows = np.concatenate(parts + ([self.z] if gate else []), axis=1)
        self.ld = u.up_to(self.rows.shape[1], 64)
        self.rows = u.padded(self.rows, self.ld)
        eps, self.lam, self.diff = 1e-3, 0.45, 0.35
        self.eps = eps
        conv = np.zeros((max(taps, 1), self.channels), np.float32)
        x = self.rows[:, :self.channels].astype(f64)
        if taps:
            conv = (g.standard_normal((taps, self.channels)) / np.sqrt(taps)).astype(np.float32)
            x = so.short_convolution(x, conv.T.astype(f64))
        self.convolved = x
        nq, nk = heads * maps * self.dimp, kv * maps * self.dimp
        q, k = x[:, :nq].reshape(n, heads * maps, self.dimp)[..., :dim], x[:, nq:nq + nk].reshape(n, kv * maps, self.dimp)[..., :dim]
        at = nq if keys_as_values else nq + nk
        v = x[:, at:at + kv * self.vdimp].reshape(n, kv, self.vdimp)
        qw, kw = (1.0 + 0.3 * g.standard_normal(dim)).astype(np.float32), (1.0 + 0.3 * g.standard_normal(dim)).astype(np.float32)
        factor = (sharp * 0.8 / np.sqrt(dim) * (1.0 + g.random(self.cap))).astype(np.float32)
        if normed:
            q, k = so.norm_plain(q, qw.astype(f64), eps), so.norm_plain(k, kw.astype(f64), eps)
        angle = np.arange(self.cap)[:, None] * (300.0 ** (-np.arange(max(rot // 2, 1)) / max(rot // 2, 1)))
        self.cos, self.sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
        if rot:
            for a in (q, k):
                c, s, e, o = self.cos[:n, None].astype(f64), self.sin[:n, None].astype(f64), a[..., :rot:2].copy(), a[..., 1:rot:2].copy()
                a[..., :rot:2], a[..., 1:rot:2] = e * c - o * s, o * c + e * s
        self.q = q * factor[:n, None, None]
        self.k, self.v = u.padded(k, self.dimp).reshape(n, kv, maps, self.dimp).transpose(1, 2, 0, 3), v.transpose(1, 0, 2)
        self.sink = g.standard_normal(heads).astype(np.float32) if sink else None
        self.far = (g.uniform(0.1, 1.2, heads).astype(np.float32), g.uniform(0.01, 2.0, heads).astype(np.float32)) if far else None
        self.cache = Cache(kv, maps, self.cap, self.dimp, self.vdimp, fill, scale)
        self.keep = [u.dev_f32(a) for a in (qw, kw, factor, self.cos, self.sin, conv)] + [u.zeros_f32(max(taps, 1), self.channels) + 99]
        p = [t.data_ptr() for t in self.keep]
        self.attn = pkg.Gqa(heads, kv, maps, dim, self.dimp, vdim, self.vdimp, self.cap, eps, self.lam, 1.0 - self.diff, p[0] if normed else 0, p[1] if normed else 0, p[2],
                            self.cache.k.data_ptr(), self.cache.v.data_ptr(), values_are_keys=int(keys_as_values), rot_dims=rot, chunk=chunk, window=window)
        if rot:
            self.attn.rope_cos, self.attn.rope_sin = p[3], p[4]
        if sink:
            self.keep.append(u.dev_f32(self.sink))
            self.attn.sink = self.keep[-1].data_ptr()
        if far:
            self.keep += [u.dev_f32(a) for a in self.far]
            self.attn.far_weight, self.attn.far_rate = self.keep[-2].data_ptr(), self.keep[-1].data_ptr()
        if taps:
            self.attn.taps, self.attn.conv, self.attn.ring = taps, p[5], p[6]

    def put(self, a):
        return u.dev_f32(a) if self.f32 else u.dev_bf16(a)

    def gated(self, rows):
        if self.gate:
            self.attn.gate = rows.data_ptr() + self.channels * rows.element_size()
            self.attn.ldgate, self.attn.gate_f32, self.attn.gate_columns = self.ld, rows.element_size() == 4, self.gate == "columns"

    def fill(self, hip, n0, n1, stream=0):
        """tokens n0 .. n1 - 1 into the cache; (rows, queries [n][heads x maps x dimp])"""
        rows, pos, n = self.put(self.rows[n0:n1]), u.dev(np.array([n0], np.int32)), n1 - n0
        self.gated(rows)
        q = (u.zeros_f32 if self.f32 else u.zeros_bf16)(n, self.heads * self.maps * self.dimp)
        hip.kv8_rows_dev(self.attn, self.cache.ks, self.cache.vs, rows, self.ld, self.f32, pos, n, q, q.shape[1], stream=stream)
        if self.taps:
            hip.conv_keep_dev(rows, self.ld, self.f32, self.channels, self.taps, self.keep[6], pos, n, stream=stream)
        return rows, q

    def step(self, hip, i, queries_only=False, out=None, scratch=None, stream=0):
        """token i from its convolved row, as the product ahead of it leaves it"""
        row = self.rows[i].astype(np.float32).copy()
        row[:self.channels] = self.convolved[i]
        row, pos = u.dev_f32(row), u.dev(np.array([i], np.int32))
        self.gated(row)
        taps, self.attn.taps, self.attn.queries_only = self.attn.taps, 0, int(queries_only)
        scratch = u.zeros_f32(hip.gqa_scratch_bytes(self.heads, self.maps, self.vdimp, 1) // 4) if scratch is None else scratch
        out = u.zeros_f32(1, self.heads * self.vdimp) if out is None else out
        hip.kv8_step_dev(self.attn, self.cache.ks, self.cache.vs, row, pos, scratch, stream=stream)
        hip.gqa_merge_dev(self.attn, pos, 0, 1, scratch, out, self.heads * self.vdimp, False, stream=stream)
        self.attn.taps, self.attn.queries_only = taps, 0
        return out

    def prompt(self, hip, q, n0, n1, split=True, out=None, stream=0):
        n, no = n1 - n0, self.heads * self.vdimp
        out = u.zeros_bf16(n, no) if out is None else out
        apart = self.maps == 2 and max(self.dimp, self.vdimp) > 128  # (which the call does not do without)
        size = hip.kv8_prefill_scratch_bytes(self.attn, n1, n) if split or apart else 0
        scratch = u.zeros_f32(size // 4) if size else None
        hip.kv8_prefill_dev(self.attn, self.cache.ks, self.cache.vs, q, q.shape[1], n1, n, out, no, scratch, size, stream=stream)
        return out

    def want(self, q, n0, held=None):
        """the attention's output for queries q [n][heads x maps][dim] at positions n0 .. over what the cache holds"""
        k, v = held if held is not None else self.cache.held()
        n, group = len(q), self.heads // self.kv
        out = np.zeros((n, self.heads, self.vdimp))
        self.gain = np.ones(self.heads)
        j = np.arange(self.cap)
        for i in range(n):
            p = n0 + i
            first = p // self.chunk * self.chunk if self.chunk else 0
            if self.window:
                first = max(first, p - self.window + 1)
            for h in range(self.heads):
                maps = []
                for m in range(self.maps):
                    s = k[h // group, m, first:p + 1, :self.dim] @ q[i, h * self.maps + m].astype(f64)
                    if self.far:
                        s = s - f64(self.far[0][h]) * np.log1p(f64(self.far[1][h]) * (p - j[first:p + 1]))
                    top = max(s.max(), f64(self.sink[h])) if self.sink is not None else s.max()
                    e = np.exp(s - top)
                    maps.append(e @ v[h // group, first:p + 1] / (e.sum() + (np.exp(f64(self.sink[h]) - top) if self.sink is not None else 0.0)))
                o = maps[0]
                if self.maps == 2:
                    o = maps[0] - self.lam * maps[1]
                    # errors of e |a1| and e |a2| are (|a1| + lambda |a2|) / |a1 - lambda a2| times e of the difference, and of what it is divided by its own length
                    self.gain[h] = max(self.gain[h], (np.linalg.norm(maps[0]) + self.lam * np.linalg.norm(maps[1])) / np.linalg.norm(o))
                    o = o / np.sqrt((o * o).sum() / self.vdim + self.eps) * (1.0 - self.diff)
                out[i, h] = o
        if self.gate:
            out *= so.sigmoid(self.z[n0:n0 + n].astype(f64)).reshape(n, self.heads, -1)
        return out

    def check(self, got, want, tol, rounding=0.0):
        """tol: of a map's output, and what a difference of two makes of it; rounding: of the output behind that"""
        got = u.host(got).reshape(want.shape)
        for h in range(self.heads):
            e = u.rms_error(got[:, h, :self.vdim], want[:, h, :self.vdim])
            assert e < tol * self.gain[h] + rounding, (h, e)
        assert not got[..., self.vdim:].any()
