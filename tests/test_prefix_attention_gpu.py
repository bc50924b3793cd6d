"""cngpt_cuda_prefix_attention against its definition in 64 bits."""
import math

import numpy as np
import pytest
import torch

from cngpt_b200 import abi

pytestmark = pytest.mark.gpu
EPS = float(torch.finfo(torch.float32).eps) / 2


class Case:
    """Inputs on the device, with pitches wider than the rows and NaN between
    them and behind every sequence's suffix, where nothing may be read."""

    def __init__(self, B, H, Hk, hs, P, S, lens=None, seed=0, pad=0, qscale=1.5):
        self.B, self.H, self.Hk, self.hs, self.P, self.S = B, H, Hk, hs, P, S
        g = torch.Generator(device="cuda").manual_seed(seed)
        n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.scale = 1.0 / math.sqrt(hs)
        self.ldq, self.ldp, self.lds, self.ldo = H * hs + pad, Hk * hs + pad, Hk * hs + 2 * pad, H * hs + 3 * pad
        self.stride = S * self.lds + 5 * pad
        nan = lambda *s: torch.full(s, math.nan, device="cuda")  # noqa: E731
        self.q, self.pk, self.pv = nan(B, self.ldq), nan(max(P, 1), self.ldp), nan(max(P, 1), self.ldp)
        self.sk, self.sv = nan(B, max(self.stride, 1)), nan(B, max(self.stride, 1))
        self.q[:, : H * hs] = n(B, H * hs) * qscale
        if P:
            self.pk[:, : Hk * hs], self.pv[:, : Hk * hs] = n(P, Hk * hs), n(P, Hk * hs)
        self.lens = np.full(B, S) if lens is None else np.asarray(lens)
        if S:
            for b in range(B):
                c = int(np.clip(self.lens[b], 0, S))
                for t in (self.sk, self.sv):
                    t[b, : S * self.lds].view(S, self.lds)[:c, : Hk * hs] = n(c, Hk * hs)
        self.len = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        self.out = torch.full((B + 1, self.ldo), 77.0, device="cuda")

    def call(self, lib, ws=None):
        n = lib.cngpt_cuda_prefix_attention_workspace(self.B, self.H, self.Hk, self.hs, self.P, self.S)
        if ws is None:
            ws = torch.full((max(n, 16) // 4 + 8,), math.nan, device="cuda")  # its contents do not matter
        p = lambda t, on: t.data_ptr() if on else None  # noqa: E731
        st = lib.cngpt_cuda_prefix_attention(
            self.q.data_ptr(), self.ldq, p(self.pk, self.P), p(self.pv, self.P), self.ldp, self.P, p(self.sk, self.S),
            p(self.sv, self.S), self.lds, self.stride, p(self.len, self.S), self.S, self.out.data_ptr(), self.ldo, self.B,
            self.H, self.Hk, self.hs, self.scale, ws.data_ptr(), n)
        abi.check(lib, st, "prefix_attention")
        return ws

    def result(self, lib):
        self.ws = self.call(lib)
        abi.check(lib, lib.cngpt_cuda_check(), "sync")
        assert (self.out[self.B] == 77.0).all() and (self.out[:, self.H * self.hs:] == 77.0).all()
        return self.out[: self.B, : self.H * self.hs].view(self.B, self.H, self.hs)

    def reference(self):
        """(output, largest sum of |q k| scale, sum of p |v|) in 64 bits."""
        B, H, Hk, hs, P, S = self.B, self.H, self.Hk, self.hs, self.P, self.S
        out = torch.zeros(B, H, hs, dtype=torch.float64, device="cuda")
        mag = torch.zeros_like(out)
        big = 0.0
        for b in range(B):
            c = int(np.clip(self.lens[b], 0, S))
            parts = [(self.pk[:P], self.pv[:P])] if P else []
            if c:
                parts.append(tuple(t[b, : S * self.lds].view(S, self.lds)[:c] for t in (self.sk, self.sv)))
            if not parts:
                continue
            k, v = (torch.cat([q[i][:, : Hk * hs].double() for q in parts]).view(-1, Hk, hs)
                    .repeat_interleave(H // Hk, 1) for i in (0, 1))
            q = self.q[b, : H * hs].double().view(H, hs)
            s = torch.einsum("hd,jhd->hj", q, k) * float(np.float32(self.scale))
            big = max(big, float((torch.einsum("hd,jhd->hj", q.abs(), k.abs()) * self.scale).nan_to_num(0.0, 0.0, 0.0).max()))
            m = s.max(1, keepdim=True).values
            e = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
            z = e.sum(1, keepdim=True)
            e = e / torch.where(z == 0, torch.ones_like(z), z)
            v = torch.where(e.T[:, :, None] == 0, torch.zeros_like(v), v)  # weight 0 takes nothing, whatever stands there
            out[b] = torch.einsum("hj,jhd->hd", e, v)
            mag[b] = torch.einsum("hj,jhd->hd", e, v.abs())
        return out, big, mag

    def check(self, lib, rel=None):
        got = self.result(lib).double()
        ref, big, mag = self.reference()
        # A score is a sum of hs products: one rounding each, two more in the
        # split of a product into three (2^-22, four roundings), so (hs + 8)
        # roundings of the sum of |q k|; the exponent's scaling adds 3 of the
        # score. An error d of the scores changes a weight by at most 2 d. The
        # sums over keys run in chains of at most 512 terms, and at most 64
        # partial results are joined with 4 roundings each.
        tol = 2 * (self.hs + 8 + 6) * EPS * big + (512 + 4 * 64) * EPS if rel is None else rel
        off = (got - ref).abs()
        assert (off <= tol * mag + 1e-37).all(), (float((off / mag.clamp(min=1e-30)).max()), tol)
        # in the norm, where roundings do not all add up, a tenth of that is ample
        assert float(off.norm()) <= (0.1 * tol if rel is None else rel) * float(mag.norm()) + 1e-37
        return got


@pytest.mark.parametrize("P,S", [(1, 0), (0, 1), (1, 1), (63, 1), (64, 64), (65, 5), (127, 130), (768, 255), (1000, 33),
                                 (0, 700), (4099, 0), (9000, 513)])
@pytest.mark.parametrize("B", [1, 3, 16])
def test_lengths(lib, cuda, P, S, B):
    Case(B, 12, 12, 64, P, S, seed=P + S).check(lib)


@pytest.mark.parametrize("H,Hk,hs", [(1, 1, 1), (3, 3, 8), (2, 1, 7), (4, 2, 16), (6, 6, 20), (8, 2, 32), (5, 5, 33), (4, 4, 48),
                                     (25, 25, 64), (16, 4, 64), (12, 1, 64), (6, 2, 80), (4, 4, 96), (24, 6, 128), (3, 1, 131),
                                     (2, 2, 200), (4, 2, 256)])
def test_head_layouts(lib, cuda, H, Hk, hs):
    for B, P, S in ((1, 70, 3), (5, 130, 40), (17, 300, 9)):
        Case(B, H, Hk, hs, P, S, seed=hs).check(lib)


@pytest.mark.parametrize("H,Hk,hs", [(1, 1, 1), (3, 3, 8), (2, 1, 7), (4, 2, 16), (6, 6, 20), (8, 2, 32), (5, 5, 33), (25, 25, 64),
                                     (12, 1, 64), (6, 2, 80), (24, 6, 128), (3, 1, 131), (4, 2, 256)])
def test_head_layouts_beyond_one_block(lib, cuda, H, Hk, hs):
    for B, P, S in ((1, 385, 3), (5, 449, 40), (17, 321, 70)):
        Case(B, H, Hk, hs, P, S, lens=[(7 * i) % (S + 1) for i in range(B)], seed=H).check(lib)


@pytest.mark.parametrize("P,S", [(1, 0), (0, 1), (1, 1), (63, 1), (64, 64), (65, 5), (127, 130), (384, 0), (383, 1), (384, 1),
                                 (0, 385)])
@pytest.mark.parametrize("B", [2, 25])
def test_lengths_on_both_sides_of_one_block(lib, cuda, P, S, B):
    Case(B, 12, 12, 64, P, S, lens=np.arange(B) % (S + 1), seed=P + S).check(lib)


@pytest.mark.parametrize("pad", [1, 2, 4])
def test_pitches_beyond_one_block(lib, cuda, pad):
    Case(6, 4, 4, 64, 400, 50, lens=[0, 50, 3, 17, 49, 1], pad=pad).check(lib)
    Case(3, 4, 2, 20, 377, 50, lens=[0, 50, 3], pad=pad).check(lib)


@pytest.mark.parametrize("B", [2, 7, 8, 9, 15, 17, 31, 32, 33, 63, 64, 65, 100, 129, 200])
def test_batches(lib, cuda, B):
    Case(B, 2, 2, 64, 515, 20, seed=B).check(lib)
    Case(B, 6, 2, 64, 130, 70, lens=np.arange(B) % 71, seed=B).check(lib)


def test_ragged_suffixes_with_empty_ones(lib, cuda):
    rng = np.random.default_rng(0)
    lens = rng.integers(0, 301, 40)
    lens[[0, 5, 39]] = 0
    lens[[1, 6]] = 300
    lens[7], lens[8] = -4, 999  # clamped
    Case(40, 12, 12, 64, 333, 300, lens=lens, seed=1).check(lib)


def test_sequences_without_keys_get_zeros(lib, cuda):
    lens = np.array([0, 3, 0, 9, -1])
    c = Case(5, 4, 4, 64, 0, 9, lens=lens)
    got = c.check(lib)
    assert (got[[0, 2, 4]] == 0).all()
    got = Case(3, 4, 2, 32, 0, 0).result(lib)
    assert (got == 0).all()


@pytest.mark.parametrize("pad", [1, 2, 4, 12])
def test_pitches_and_alignment(lib, cuda, pad):
    Case(6, 4, 4, 64, 200, 50, lens=[0, 50, 3, 17, 49, 1], pad=pad).check(lib)
    Case(3, 4, 2, 20, 77, 50, lens=[0, 50, 3], pad=pad).check(lib)


def test_unaligned_base_addresses(lib, cuda):
    c = Case(4, 4, 4, 64, 150, 30, seed=3)
    for name in ("q", "pk", "pv", "sk", "sv"):
        t = getattr(c, name)
        flat = torch.full((t.numel() + 1,), math.nan, device="cuda")
        flat[1:] = t.reshape(-1)
        setattr(c, name, flat[1:].view(t.shape))
    c.check(lib)


@pytest.mark.parametrize("q", [0.0, 30.0])
def test_flat_and_sharp_softmax(lib, cuda, q):
    Case(9, 4, 4, 64, 700, 100, qscale=q, seed=4).check(lib)


def test_keys_of_very_low_scores(lib, cuda):
    """Finite keys so low that their weight is 0 beside the others, also whole
    tiles of them, and sequences that see no other key."""
    c = Case(4, 2, 2, 64, 400, 40, seed=5)
    c.q[:, : 2 * 64] = c.q[:, : 2 * 64].abs() + 0.1
    c.pk[:210, :128] = -1e30
    c.pk[300, :128] = -1e36
    c.sk[1, : 40 * c.lds].view(40, c.lds)[:, :128] = -1e34
    ref, _, mag = c.reference()
    got = c.result(lib).double()
    # the weights of the other keys are as exact as without the low ones
    clean = 2 * 78 * EPS * float(((c.q[:, :128].abs().amax()) * 64 * 4.5 / 8)) + 768 * EPS
    assert ((got - ref).abs() <= clean * mag).all()
    c.pk[:, :128] = -1e30  # equal scores alone in the prefix, sequence 1 sees nothing above them
    ref, _, mag = c.reference()
    got = c.result(lib).double()
    assert torch.isfinite(got).all()
    assert ((got - ref)[[0, 2, 3]].abs() <= clean * mag[[0, 2, 3]]).all()


def test_tf32_mode(lib, cuda):
    """One TF32 pass: operands are cut to 10 bits, 2^-10 relative each."""
    lib.cngpt_cuda_set_precision(abi.PREC_TF32)
    try:
        c = Case(16, 12, 12, 64, 500, 40, seed=6)
        _, big, _ = c.reference()
        c.check(lib, rel=2 * 2 * 2.0 ** -10 * big + 3 * 2.0 ** -10)
    finally:
        lib.cngpt_cuda_set_precision(abi.PREC_3XTF32)


def test_fp32_mode(lib, cuda):
    lib.cngpt_cuda_set_precision(abi.PREC_FP32)
    try:
        Case(16, 12, 12, 64, 500, 40, seed=7).check(lib)
    finally:
        lib.cngpt_cuda_set_precision(abi.PREC_3XTF32)


def test_long_cache_offsets_beyond_32_bits(lib, cuda):
    """Suffixes that start beyond 2^31 floats."""
    B, H, hs, S = 3, 2, 64, 17
    c = Case(B, H, H, hs, 100, S, lens=[17, 9, 17], seed=8)
    stride = (1 << 30) + 3
    sk, sv = c.sk, c.sv
    big = [torch.empty(2 * stride + c.stride + 8, device="cuda") for _ in range(2)]
    for t, s in zip(big, (sk, sv)):
        for b in range(B):
            t[b * stride: b * stride + c.stride] = s[b]
    old = c.stride
    c.sk, c.sv, c.stride = big[0], big[1], stride
    got = c.result(lib).clone()
    c.sk, c.sv, c.stride = sk, sv, old
    ref, bigv, mag = c.reference()
    assert ((got.double() - ref).abs() <= (2 * 78 * bigv + 768) * EPS * mag).all()


def test_one_sequence_is_plain_decode_attention(lib, cuda):
    """Without a suffix and with one sequence: the same as the causal kernel's
    last row over the same keys."""
    T, Cm, H = 200, 256, 4
    qkv = torch.randn(T, 3 * Cm, device="cuda")
    out = torch.empty(T, Cm, device="cuda")
    abi.check(lib, lib.cngpt_cuda_attention_fwd(qkv.data_ptr(), out.data_ptr(), None, 1, T, Cm, H))
    n = lib.cngpt_cuda_prefix_attention_workspace(1, H, H, 64, T, 0)
    ws, o = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda"), torch.empty(Cm, device="cuda")
    f = 4
    abi.check(lib, lib.cngpt_cuda_prefix_attention(qkv.data_ptr() + f * (T - 1) * 3 * Cm, 3 * Cm, qkv.data_ptr() + f * Cm,
                                                   qkv.data_ptr() + f * 2 * Cm, 3 * Cm, T, None, None, 0, 0, None, 0,
                                                   o.data_ptr(), Cm, 1, H, H, 64, 0.125, ws.data_ptr(), n))
    abi.check(lib, lib.cngpt_cuda_check())
    assert float((o - out[T - 1]).abs().max()) <= 1e-5 * float(out[T - 1].abs().max())


def test_repeatable_and_two_graphs_with_their_own_workspaces(lib, cuda):
    a, b = Case(16, 12, 12, 64, 768, 100, seed=9), Case(5, 4, 2, 64, 1200, 7, seed=10)
    ra, rb = a.result(lib).clone(), b.result(lib).clone()
    assert torch.equal(ra, a.result(lib)) and torch.equal(rb, b.result(lib))
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, keep = [], []
    try:
        for c, s in zip((a, b), side):
            n = lib.cngpt_cuda_prefix_attention_workspace(c.B, c.H, c.Hk, c.hs, c.P, c.S)
            ws = torch.empty(max(n, 16) // 4 + 4, device="cuda")
            g = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(g, stream=s):
                lib.cngpt_cuda_set_stream(s.cuda_stream)
                c.call(lib, ws)
            graphs.append(g)
            keep.append(ws)
        a.out.fill_(77.0)
        b.out.fill_(77.0)
        torch.cuda.synchronize()
        for _ in range(4):
            for g, s in zip(graphs, side):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for c, r in ((a, ra), (b, rb)):
            assert torch.equal(c.out[: c.B, : c.H * c.hs].view(c.B, c.H, c.hs), r)
    finally:
        lib.cngpt_cuda_set_stream(None)


def test_small_workspace_is_refused(lib, cuda):
    c = Case(16, 12, 12, 64, 768, 100)
    n = lib.cngpt_cuda_prefix_attention_workspace(c.B, c.H, c.Hk, c.hs, c.P, c.S)
    if n == 0:
        return
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    for at, size in ((ws.data_ptr(), n - 1), (ws.data_ptr() + 4, n), (None, n)):
        st = lib.cngpt_cuda_prefix_attention(c.q.data_ptr(), c.ldq, c.pk.data_ptr(), c.pv.data_ptr(), c.ldp, c.P,
                                             c.sk.data_ptr(), c.sv.data_ptr(), c.lds, c.stride, c.len.data_ptr(), c.S,
                                             c.out.data_ptr(), c.ldo, c.B, c.H, c.Hk, c.hs, c.scale, at, size)
        assert st == abi.ERR_ARG
    lib.cngpt_cuda_clear_status()
