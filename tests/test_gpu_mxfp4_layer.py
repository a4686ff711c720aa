"""The 4-bit operators together, as an attention layer's decoding steps run them: the
activations packed and multiplied with packed weights, Q and K turned, K and V written into
a 4-bit paged cache, one new token's attention over it, and the output projection.  Each
stage is checked against 64 bits from what the stage before it gave, so that each has its
own bound: a product half a bf16 step and its fp32 sums, a turn the same, the cache's bytes
exact, and attention that of test_gpu_paged_attention.py."""
from __future__ import annotations

import numpy as np
import pytest

import mxfp4_ref as ref

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV_HEADS, D, PAGE, COLS = 384, 8, 2, 64, 16, 8


def _host(x):
    return x.double().cpu().numpy()


def _product_bound(a, b, want):
    return np.abs(want) * 2.0 ** -8 * 1.01 + (np.abs(a) @ np.abs(b).T) * a.shape[1] * 2.0 ** -24


class Layer:
    def __init__(self, torch, seed, seqs):
        from fe2o3_amd import kernels as k
        self.k, self.torch, self.seqs = k, torch, seqs
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        width = (HEADS + 2 * KV_HEADS) * D
        self.w_qkv = self.weight(width, HIDDEN)
        self.w_out = self.weight(HIDDEN, HEADS * D)
        pages = seqs * COLS + 2
        self.arrays = [torch.zeros(pages, PAGE, KV_HEADS, D // 2, dtype=torch.uint8, device="cuda")
                       for _ in "kv"]
        self.scales = [torch.full((pages, KV_HEADS, PAGE, D // 32), 255, dtype=torch.uint8,
                                  device="cuda") for _ in "kv"]  # NaN where no row is
        self.cache = k.KvCache(*self.arrays, *self.scales)
        self.table = torch.randperm(pages, generator=self.gen, device="cuda")[:seqs * COLS].reshape(
            seqs, COLS).to(torch.int32)
        table, self.scale = k.rotary_frequencies(D, factor=4.0, schedule="by_turns")
        self.freq_host, self.freq = table, torch.from_numpy(table).cuda()
        bf = dict(dtype=torch.bfloat16, device="cuda")
        self.x = torch.zeros(seqs, HIDDEN, **bf)
        self.qkv = torch.empty(seqs, HEADS + 2 * KV_HEADS, D, **bf)
        self.q = torch.empty(seqs, HEADS, D, **bf)
        self.key = torch.empty(seqs, KV_HEADS, D, **bf)
        self.attended = torch.empty(seqs, HEADS, D, **bf)
        self.lse = torch.empty(seqs, HEADS, device="cuda")
        self.out = torch.empty(seqs, HIDDEN, **bf)
        self.positions = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        self.lengths = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        self.slots = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        self.a_x, self.a_o = self.packed(seqs, HIDDEN), self.packed(seqs, HEADS * D)
        self.work = torch.empty(k.paged_attention_workspace_bytes(HEADS, KV_HEADS, D),
                                dtype=torch.uint8, device="cuda")

    def packed(self, rows, cols):
        return [self.torch.zeros(s, dtype=self.torch.uint8, device="cuda")
                for s in self.k.mxfp4_shapes(rows, cols)]

    def weight(self, rows, cols):
        w = self.torch.randn(rows, cols, generator=self.gen, device="cuda") * cols ** -0.5
        arrays = self.packed(rows, cols)
        self.k.quantize_mxfp4(w, *arrays)
        return arrays

    def step(self, stream):
        k, s = self.k, dict(stream=stream, sync=False)
        k.quantize_mxfp4(self.x, *self.a_x, **s)
        k.gemm_mxfp4_nt(*self.a_x, *self.w_qkv, self.qkv.view(self.seqs, -1), **s)
        k.rotary(self.qkv[:, :HEADS], self.qkv[:, HEADS:HEADS + KV_HEADS], self.positions,
                 self.freq, q_out=self.q, k_out=self.key, scale=self.scale, **s)
        k.kv_cache_write(self.cache, self.key, self.values(), self.slots, **s)
        k.paged_attention_decode(self.cache, self.q, self.table, self.lengths, self.attended,
                                 self.lse, self.work, max_length=COLS * PAGE, scale=D ** -0.5, **s)
        k.quantize_mxfp4(self.attended.view(self.seqs, -1), *self.a_o, **s)
        k.gemm_mxfp4_nt(*self.a_o, *self.w_out, self.out, **s)

    def values(self):
        # dense rows of V's own, with K's strides
        self.v = self.qkv[:, HEADS + KV_HEADS:].contiguous()
        return self.v

    def place(self, positions):
        """Positions, lengths and slots of the step's tokens; -1: a padded row."""
        at = np.asarray(positions)
        table = self.table.cpu().numpy()
        seq = np.arange(self.seqs)
        slot = np.where(at < 0, -1, table[seq, np.maximum(at, 0) // PAGE] * PAGE + at % PAGE)
        for name, value in (("positions", at), ("lengths", np.maximum(at + 1, 0)), ("slots", slot)):
            getattr(self, name).copy_(self.torch.from_numpy(value.astype(np.int32)))

    def check(self, positions, history):
        """Every stage of the last step; history[s]: K and V rows in 64 bits so far."""
        x = ref.unpack(*(v.cpu().numpy() for v in self.a_x))
        want_q, want_s = ref.pack(self.x.float().cpu().numpy())
        assert np.array_equal(self.a_x[0].cpu().numpy(), want_q)
        w = ref.unpack(*(v.cpu().numpy() for v in self.w_qkv))
        want = x @ w.T
        got = _host(self.qkv).reshape(self.seqs, -1)
        assert np.all(np.abs(got - want) <= _product_bound(x, w, want))
        for name, rows, out in (("q", self.qkv[:, :HEADS], self.q),
                                ("k", self.qkv[:, HEADS:HEADS + KV_HEADS], self.key)):
            r = _host(rows)
            t = np.maximum(positions, 0)[:, None, None] * self.freq_host
            c, s = np.cos(t) * self.scale, np.sin(t) * self.scale
            a, b = r[..., :D // 2], r[..., D // 2:]
            want = np.concatenate([a * c - b * s, b * c + a * s], -1)
            size = np.abs(np.concatenate([a, a], -1)) + np.abs(np.concatenate([b, b], -1))
            live = np.asarray(positions) >= 0
            off = np.abs(_host(out) - want)
            assert np.all(off[live] <= (np.abs(want) * 2.0 ** -8 * 1.01
                                        + size * self.scale * 2.0 ** -21)[live]), name
        for s, at in enumerate(positions):
            if at < 0:
                assert not _host(self.attended)[s].any() and np.all(
                    np.isneginf(self.lse[s].cpu().numpy()))
                continue
            new = []
            for rows in (self.key, self.v):
                blocks = rows[s].float().cpu().numpy().reshape(KV_HEADS, D // 32, 32)
                byte = ref.scale_bytes(blocks)
                new.append(ref.values(ref.codes(blocks, byte), byte).reshape(KV_HEADS, D))
            history[s].append(new)
            kk = np.stack([h[0] for h in history[s]])
            vv = np.stack([h[1] for h in history[s]])
            q = _host(self.q)[s].reshape(KV_HEADS, -1, D)
            for h in range(KV_HEADS):
                sc = q[h] @ kk[:, h].T * D ** -0.5
                p = np.exp(sc - sc.max(-1, keepdims=True))
                p /= p.sum(-1, keepdims=True)
                want, mean = p @ vv[:, h], p @ np.abs(vv[:, h])
                score = (D + 4) * 2.0 ** -24 * (np.abs(q[h]) @ np.abs(kk[:, h]).T).max() * D ** -0.5
                bound = mean * (2.0 ** -8 * 1.01 + 2 * score + 2.0 ** -20) + np.abs(want) * 2.0 ** -8
                got = _host(self.attended)[s].reshape(KV_HEADS, -1, D)[h]
                assert np.all(np.abs(got - want) <= bound)
        o = ref.unpack(*(v.cpu().numpy() for v in self.a_o))
        w = ref.unpack(*(v.cpu().numpy() for v in self.w_out))
        want = o @ w.T
        assert np.all(np.abs(_host(self.out) - want) <= _product_bound(o, w, want))


@pytest.mark.parametrize("captured", [False, True])
def test_decoding_steps(gpu, captured):
    torch = pytest.importorskip("torch")
    layer = Layer(torch, 11, 4)
    history = [[] for _ in range(4)]
    side = torch.cuda.Stream()
    graph = None
    for turn in range(6):
        # one sequence joins later, one row is padding
        positions = np.array([turn, turn, turn - 2 if turn >= 2 else -1, -1])
        layer.x.copy_(torch.randn(layer.x.shape, generator=layer.gen, device="cuda"))
        layer.place(positions)
        torch.cuda.synchronize()
        if not captured:
            layer.step(None)
        else:
            if graph is None:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=side):
                    layer.step(side)
            graph.replay()
        torch.cuda.synchronize()
        layer.check(positions, history)


def test_two_layers_at_once(gpu):
    """Steps of two layers on two streams, each with its own scratch: the bits of the
    same steps one after the other."""
    torch = pytest.importorskip("torch")
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for together in (True, False):
        layers = [Layer(torch, seed, 4) for seed in (5, 6)]
        got = []
        for turn in range(3):
            for layer in layers:
                layer.x.copy_(torch.randn(layer.x.shape, generator=layer.gen, device="cuda"))
                layer.place(np.full(4, turn))
            torch.cuda.synchronize()
            for layer, stream in zip(layers, streams):
                with torch.cuda.stream(stream if together else torch.cuda.default_stream()):
                    layer.step(stream if together else None)
                if not together:
                    torch.cuda.synchronize()
            torch.cuda.synchronize()
            got += [t.clone() for layer in layers for t in (layer.out, layer.lse, layer.attended)]
        results.append(got)
    assert all(torch.equal(a, b) for a, b in zip(*results))
