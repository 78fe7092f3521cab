"""The operators between a block's linear layers as a model uses them: one behind the other, on streams, in graphs, from threads; what they refuse."""

import math
import threading

import pytest
import torch

import test_gpu_gated_norm as norm_test
import test_gpu_rotary_axes as rotary_test
import test_gpu_self_attention as attention_test
from conftest import announce

pytestmark = pytest.mark.gpu


class Block:
    """Images of different sizes and their prompts, packed: norm and modulation, 8-bit QKV projection, rotation, attention, 8-bit projection, gate, residual and the
    next norm."""

    def __init__(self, dev, dtype, lens, H=6, Hkv=2, D=64, K=384, causal=False, seed=0):
        from nunchaku_amd.models import W8A8Linear

        g = torch.Generator().manual_seed(seed)
        rand = lambda *s, scale=1.0: (scale * torch.randn(*s, generator=g)).to(dtype).to(dev)  # noqa: E731
        self.H, self.Hkv, self.D, self.causal, self.axes = H, Hkv, D, causal, (16, 24, 24)
        total, S = sum(lens), len(lens)
        self.stream, self.mod = rand(total, K), rand(S, 3 * K, scale=0.3)
        self.pos = torch.randint(0, 100, (total, 3), generator=g, dtype=torch.int32).to(dev)
        self.cu = attention_test.offsets(lens).to(dev)
        self.wq, self.wk = (1 + rand(D, scale=0.1) for _ in range(2))
        torch.manual_seed(seed)
        self.qkv = W8A8Linear.from_linear(torch.nn.Linear(K, (H + 2 * Hkv) * D, dtype=dtype)).to(dev)
        self.proj = W8A8Linear.from_linear(torch.nn.Linear(H * D, K, dtype=dtype)).to(dev)

    def __call__(self):
        from nunchaku_amd import ops

        gate, scale, shift = self.mod.chunk(3, 1)
        x, _ = ops.gated_norm(self.stream, norm="layer", scale=scale, shift=shift, cu_seqlens=self.cu)
        q, k, v = (t.unflatten(-1, (-1, self.D)) for t in self.qkv(x).split([self.H * self.D, self.Hkv * self.D, self.Hkv * self.D], -1))
        rq, rk = ops.rotary_axes(q, k, self.pos, self.axes, norm_q=self.wq, norm_k=self.wk)
        o = ops.self_attention(rq, rk, v, self.cu, causal=self.causal)
        y = self.proj(o.flatten(1))
        return x, q, k, v, rq, rk, o, y, *ops.gated_norm(y, self.stream, "layer", gate=gate, scale=scale, shift=shift, cu_seqlens=self.cu)

    def check(self, results):
        """Each operator's result against the oracle on what it was given."""
        x, q, k, v, rq, rk, o, y, x2, h = (t.cpu() for t in results)
        cu = self.cu.tolist()
        entry = torch.repeat_interleave(torch.arange(len(cu) - 1), self.cu.diff().cpu())
        gate, scale, shift = (t[entry] for t in self.mod.cpu().chunk(3, 1))
        stream = self.stream.cpu()
        norm_test.check((x, None), stream, None, "layer", scale=scale, shift=shift)
        rotary_test.check(rq[None], q[None], self.pos.cpu()[None], self.axes, weight=self.wq.cpu())
        rotary_test.check(rk[None], k[None], self.pos.cpu()[None], self.axes, weight=self.wk.cpu())
        for a, b in zip(cu[:-1], cu[1:]):
            attention_test.check(o[a:b], rq[a:b], rk[a:b], v[a:b], self.causal)
        norm_test.check((x2, h), y, stream, "layer", gate=gate, scale=scale, shift=shift)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
def test_a_block(dev, dtype, causal):
    announce(f"block {dtype} {causal}")
    block = Block(dev, dtype, [257, 77, 1, 400], causal=causal)
    block.check(block())


def test_a_block_in_graphs_and_on_a_stream(dev):
    """Two captured graphs replayed in turn, eager calls and a side stream between; inputs, positions and lengths change."""
    announce("block in graphs")
    blocks = [Block(dev, torch.bfloat16, lens, seed=i, causal=i == 1) for i, lens in enumerate(([300, 20, 64], [5, 900]))]
    graphs, outs = [], []
    for b in blocks:
        b()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(b())
        graphs.append(g)
    side = torch.cuda.Stream()
    for turn in range(4):
        for b in blocks:
            b.stream.mul_(-0.8)
            b.pos.add_(turn)
            b.cu[1:-1] += 1 - 2 * (turn % 2)
        eager = [b() for b in blocks]
        for o in outs:
            for t in o:
                t.zero_()
        for g in graphs if turn % 2 else graphs[::-1]:
            g.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            beside = [b() for b in blocks]
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(a, c) for x, y, z in zip(outs, eager, beside) for a, b, c in zip(x, y, z))
    for b, o in zip(blocks, outs):
        b.check(o)


def test_single_tokens_in_graphs(dev):
    """New tokens over long caches, the keys in parts: workspaces are the calls' own, lengths grow between the replays."""
    from nunchaku_amd.ops import self_attention

    announce("single tokens in graphs")
    sets = []
    for i in range(2):
        q, k, v = (attention_test.rand(*s, dtype=torch.bfloat16, seed=10 * i + j).to(dev) for j, s in enumerate([(4, 8, 128), (2, 5000 + i, 2, 128), (2, 5000 + i, 2, 128)]))
        sets.append((q, k, v, torch.tensor([0, 1 + 2 * i, 4], dtype=torch.int32, device=dev), None, torch.tensor([4000, 9], dtype=torch.int32, device=dev), True))
    graphs, outs = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(self_attention(*s))
        graphs.append(g)
    for turn in range(4):
        for s in sets:
            s[0].mul_(-0.9)
            s[5].add_(1 + 40 * turn)
        eager = [self_attention(*s) for s in sets]
        for g in graphs if turn % 2 else graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))
    for s, o in zip(sets, outs):
        cu, n = s[3].tolist(), s[5].tolist()
        for i in range(2):
            attention_test.check(o[cu[i]:cu[i + 1]], s[0][cu[i]:cu[i + 1]].cpu(), s[1][i, :n[i]].cpu(), s[2][i, :n[i]].cpu(), True)


def test_calls_from_several_threads(dev):
    announce("threads")
    blocks = [Block(dev, torch.bfloat16, [100 + 50 * i, 3], seed=i, causal=bool(i % 2)) for i in range(4)]
    want = [b() for b in blocks]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(4):
                    got[i] = blocks[i]()
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001 (reported below, in the test's own thread)
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))


def test_offsets_beyond_32_bits(dev):
    """Rows, tokens and batch entries more than 2^32 bytes into their tensors."""
    from nunchaku_amd.ops import gated_norm, rotary_axes, self_attention

    announce("offsets beyond 32 bits")
    far = 2**31 + 2**20
    big = torch.empty(2 * far, dtype=torch.bfloat16, device=dev)  # 8 GiB
    x, res = (norm_test.rand(2, 1024, dtype=torch.bfloat16, seed=i) for i in range(2))
    parts = [big.as_strided((2, 1024), (far, 1), 2048 * i) for i in range(2)]
    for p, t in zip(parts, (x, res)):
        p.copy_(t)
    norm_test.check(gated_norm(parts[0], parts[1], out=parts[0], residual_out=parts[1]), x, res)
    q, k, w, pos = rotary_test.inputs(2, 3, 2, 2, 64, 1, torch.bfloat16, 1)
    gq = big.as_strided((2, 3, 2, 64), (far, 2**19, 64, 1))
    gk = big.as_strided((2, 3, 2, 64), (far, 2**19, 64, 1), 256)
    gq.copy_(q)
    gk.copy_(k)
    got = rotary_axes(gq, gk, pos.to(dev), (64,), out_q=gq, out_k=gk)
    rotary_test.check(got[0], q, pos, (64,))
    rotary_test.check(got[1], k, pos, (64,))
    for T in (3, 400):
        q, k, v = (attention_test.rand(2, n, h, 64, dtype=torch.bfloat16, seed=s) for n, h, s in ((T, 4, 1), (T + 30, 2, 2), (T + 30, 2, 3)))
        g = [big.as_strided(t.shape, (far, 2**12, 64, 1), 512 * i) for i, t in enumerate((q, k, v))]
        for a, t in zip(g, (q, k, v)):
            a.copy_(t)
        out = torch.empty_like(q, device=dev)
        self_attention(*g, causal=True, out=out)
        for b in range(2):
            attention_test.check(out[b], q[b], k[b], v[b], True)


def test_same_from_run_to_run(dev):
    from nunchaku_amd.ops import self_attention

    for lens, H, Hkv, D in (([3000, 1, 500], 8, 2, 128), ([2000], 2, 2, 72)):
        q, k, v = (attention_test.rand(sum(lens), h, D, dtype=torch.bfloat16, seed=i).to(dev) for i, h in enumerate((H, Hkv, Hkv)))
        cu = attention_test.offsets(lens).to(dev)
        first = self_attention(q, k, v, cu, causal=True)
        assert all(torch.equal(self_attention(q, k, v, cu, causal=True), first) for _ in range(5))


def test_results_carry_no_gradient(dev):
    from nunchaku_amd.ops import gated_norm, rotary_axes, self_attention

    x = torch.randn(1, 5, 2, 64, device=dev, dtype=torch.bfloat16, requires_grad=True)
    pos = torch.zeros(5, 1, dtype=torch.int32, device=dev)
    assert not any(t.requires_grad for t in (*gated_norm(x, x), *rotary_axes(x, x, pos, (64,)), self_attention(x, x, x)))


def test_norm_refusals(dev):
    from nunchaku_amd.ops import gated_norm

    x = torch.zeros(4, 6, 64, dtype=torch.bfloat16, device=dev)
    flat, v = x.view(24, 64), x[0, 0]
    cu = torch.tensor([0, 10, 24], dtype=torch.int32, device=dev)
    for call in (
        lambda: gated_norm(x[..., :60]), lambda: gated_norm(x, norm="group"), lambda: gated_norm(x, x[0]), lambda: gated_norm(x, x.half()), lambda: gated_norm(x, weight=v[:32]),
        lambda: gated_norm(x, weight=v.half()), lambda: gated_norm(x, weight=v.cpu()), lambda: gated_norm(x, gate=x[:3, 0]), lambda: gated_norm(x, gate=x[0]), lambda: gated_norm(x, scale=v.float()),
        lambda: gated_norm(x, shift=v[:32]), lambda: gated_norm(flat, cu_seqlens=cu.long()), lambda: gated_norm(x, cu_seqlens=cu), lambda: gated_norm(flat, cu_seqlens=cu[:1]),
        lambda: gated_norm(flat, gate=flat[:3], cu_seqlens=cu), lambda: gated_norm(flat, gate=flat, cu_seqlens=cu), lambda: gated_norm(x, eps=-1.0), lambda: gated_norm(x, eps=math.nan),
        lambda: gated_norm(x, x, residual_scale=math.inf), lambda: gated_norm(x, residual_out=x), lambda: gated_norm(x, out=flat), lambda: gated_norm(x, out=x.half()),
        lambda: gated_norm(x, x, out=x, residual_out=x), lambda: gated_norm(flat, out=flat[:1].expand(24, 64)), lambda: gated_norm(x.transpose(0, 1)), lambda: gated_norm(x.transpose(1, 2)),
        lambda: gated_norm(flat[:, 4:60]), lambda: gated_norm(torch.zeros(2, 32776, dtype=torch.bfloat16, device=dev)),
    ):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(NotImplementedError):
        gated_norm(x.float())
    with pytest.raises(RuntimeError, match="GPU"):
        gated_norm(x.cpu())


def test_rotary_refusals(dev):
    from nunchaku_amd.ops import rotary_axes

    q = torch.zeros(2, 5, 4, 64, dtype=torch.bfloat16, device=dev)
    p = torch.zeros(5, 2, dtype=torch.int32, device=dev)
    for call in (
        lambda: rotary_axes(q, q, p, (64,)), lambda: rotary_axes(q, q, p, (32, 34)), lambda: rotary_axes(q, q, p, (31, 33)), lambda: rotary_axes(q, q, p, (0, 64)), lambda: rotary_axes(q, q, p, ()),
        lambda: rotary_axes(q, q, p[:, :1].expand(5, 5), (8,) * 5), lambda: rotary_axes(q, q, p[:4], (32, 32)), lambda: rotary_axes(q, q, p.short(), (32, 32)), lambda: rotary_axes(q, q, p.cpu(), (32, 32)),
        lambda: rotary_axes(q, q, p, (32, 32), theta=0.0), lambda: rotary_axes(q, q, p, (32, 32), theta=(1e4,)), lambda: rotary_axes(q, q, p, (32, 32), spectrum="none"),
        lambda: rotary_axes(q, q, p, (32, 24), interleaved=False), lambda: rotary_axes(q, q[:, :4], p, (32, 32)), lambda: rotary_axes(q, q.half(), p, (32, 32)),
        lambda: rotary_axes(q, q[..., :32], p, (16, 16)), lambda: rotary_axes(q, None, p, (32, 32), norm_k=q[0, 0, 0]), lambda: rotary_axes(q, q, p, (32, 32), norm_q=q[0, 0, 0, :32]),
        lambda: rotary_axes(q, q, p, (32, 32), eps=-1.0), lambda: rotary_axes(q, q, p, (32, 32), out_q=q[:1]), lambda: rotary_axes(q, q, p, (32, 32), out_k=q[:, :1].expand(2, 5, 4, 64)),
        lambda: rotary_axes(q[..., :60], None, p, (30, 30)), lambda: rotary_axes(q.transpose(2, 3), None, p, (2, 2)), lambda: rotary_axes(q[0, 0], None, p, (32, 32)),
        lambda: rotary_axes(q[0], None, p[None].expand(2, 5, 2), (32, 32)), lambda: rotary_axes(q[:, :, :0], q, p, (32, 32)),
    ):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(NotImplementedError):
        rotary_axes(q.float(), None, p, (32, 32))
    with pytest.raises(RuntimeError, match="GPU"):
        rotary_axes(q.cpu(), None, p, (32, 32))


def test_attention_refusals(dev):
    from nunchaku_amd.ops import self_attention

    q = torch.zeros(2, 5, 4, 64, dtype=torch.bfloat16, device=dev)
    k, f = q[:, :, :2], q.flatten(0, 1)
    cu = torch.tensor([0, 3, 10], dtype=torch.int32, device=dev)
    n = torch.tensor([3, 4], dtype=torch.int32, device=dev)
    for call in (
        lambda: self_attention(q, k, q), lambda: self_attention(q, q[:, :, :3], q[:, :, :3]), lambda: self_attention(q, k[:1], k[:1]), lambda: self_attention(q, k.half(), k.half()),
        lambda: self_attention(q, k[..., :32], k[..., :32]), lambda: self_attention(f, f, f), lambda: self_attention(q, f, f), lambda: self_attention(q, q, q, cu), lambda: self_attention(f, f, f, cu.long()),
        lambda: self_attention(f, f, f, cu, cu[:2]), lambda: self_attention(f, f, f, cu, key_lengths=n), lambda: self_attention(q, k, k, key_lengths=n[:1]), lambda: self_attention(q, k, k, key_lengths=n.long()),
        lambda: self_attention(q, k, k, cu_seqlens_k=cu), lambda: self_attention(f, k[:1], k[:1], cu), lambda: self_attention(f, f, f, cu[:1]), lambda: self_attention(f, f, f, cu.cpu()),
        lambda: self_attention(q, k, k, scale=0.0), lambda: self_attention(q, k, k, scale=math.nan), lambda: self_attention(q, k, k, out=f), lambda: self_attention(q, k, k, out=q.half()),
        lambda: self_attention(q, k, k, out=q[:1].expand(2, 5, 4, 64)), lambda: self_attention(q.transpose(2, 3), k, k), lambda: self_attention(q[..., :60], k[..., :60], k[..., :60]),
        lambda: self_attention(q[..., 4:60], k[..., :56], k[..., :56]),
    ):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(NotImplementedError):
        self_attention(q.float(), k.float(), k.float())
    with pytest.raises(RuntimeError, match="GPU"):
        self_attention(q.cpu(), k.cpu(), k.cpu())


@pytest.mark.parametrize("D", [72, 128])
def test_keys_beyond_32_bits_of_many_rows(dev, D):
    """Tokens 8 MiB apart: the last keys of a sequence are more than 2^32 bytes behind its first ones."""
    from nunchaku_amd.ops import self_attention

    announce(f"keys beyond 32 bits {D}")
    T, H, token = 700, 64, 2**22
    q, k, v = (attention_test.rand(1, T, H, D, dtype=torch.bfloat16, seed=s) for s in (1, 2, 3))
    big = torch.empty(T * token, dtype=torch.bfloat16, device=dev)  # 5.9 GB
    g = [big.as_strided((1, T, H, D), (0, token, D, 1), i * H * D) for i in range(2)]
    for a, t in zip(g, (k, v)):
        a.copy_(t)
    for causal in (False, True):
        attention_test.check(self_attention(q.to(dev), *g, causal=causal)[0], q[0], k[0], v[0], causal)
