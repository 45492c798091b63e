"""The paged 4-bit cache (append with rotation, read-back, ragged decode
attention) against a plain implementation in 64 bits that decodes the page
format token by token."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
ULP = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step of the type, relative


class Oracle:
    """Keys and values of sequences in numpy: what each token is held as."""

    def __init__(self, sink, recent, dt):
        self.sink, self.recent, self.dt = sink, recent, dt
        self.k, self.v = {}, {}  # sequence -> [n, H, D] in the type, rotated
        self.ck, self.cv = {}, {}  # what the cache holds, float64

    def rnd(self, x):
        return torch.from_numpy(np.asarray(x, np.float32)).to(self.dt).float().numpy()

    def packed(self, n):
        return max(0, n - self.sink - self.recent) // 32 * 32

    def group(self, x, axis):
        """A tile quantized in groups of 32 along axis (whole axis in groups), as float64."""
        x = np.moveaxis(x.astype(np.float32), axis, -1)
        g = x.reshape(x.shape[:-1] + (-1, 32))
        with np.errstate(all="ignore"):
            top = np.abs(g).max(-1, keepdims=True)
            scale = self.rnd(top / np.float32(7))
            q = self.rnd(np.abs(g) / scale)
            c = np.rint(np.clip(np.nan_to_num(q, nan=0.0, posinf=7.0), 0, 7)) * np.sign(np.nan_to_num(g))
            good = np.isfinite(top)
            val = np.where(good, c, 0) * np.where(good, scale, np.nan).astype(np.float64)
        return np.moveaxis(val.reshape(x.shape), -1, axis)

    def append(self, b, k, v):
        """k (rotated) and v [n, H, D] in the type, as float32."""
        old = self.k[b].shape[0] if b in self.k else 0
        cat = lambda d, x: np.concatenate([d[b], x]) if b in d else x  # noqa: E731
        self.k[b], self.v[b] = cat(self.k, k), cat(self.v, v)
        self.ck[b], self.cv[b] = cat(self.ck, k.astype(np.float64)), cat(self.cv, v.astype(np.float64))
        lo, hi = self.packed(old), self.packed(self.k[b].shape[0])
        for t in range(self.sink + lo, self.sink + hi, 32):
            self.ck[b][t:t + 32] = self.group(self.k[b][t:t + 32], 2)
            self.cv[b][t:t + 32] = self.group(self.v[b][t:t + 32], 0)

    def attend(self, b, q, scale):
        """q [Hq, D] float -> out [Hq, D], lse (base 2)."""
        k, v = self.ck[b], self.cv[b]
        R = q.shape[0] // k.shape[1]
        out = np.zeros(q.shape)
        lse = np.full(q.shape[0], -np.inf)
        for h in range(q.shape[0]):
            s = k[:, h // R] @ q[h].astype(np.float64) * scale
            if len(s):
                m = s.max()
                p = np.exp(s - m)
                out[h] = p @ v[:, h // R] / p.sum()
                lse[h] = (m + np.log(p.sum())) / math.log(2)
        return out, lse


def rotate64(x, cos, sin, interleaved):
    """x [n, H, D] float32, cos / sin [n, rot / 2]: fp32 products and sums."""
    x = x.astype(np.float32)
    r = 2 * cos.shape[1]
    c, s = cos[:, None].astype(np.float32), sin[:, None].astype(np.float32)
    y = x.copy()
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    p, q = a * c - b * s, b * c + a * s
    if interleaved:
        y[..., 0:r:2], y[..., 1:r:2] = p, q
    else:
        y[..., :r // 2], y[..., r // 2:r] = p, q
    return y


def table(n, rot):
    ang = np.arange(n)[:, None] * 10000.0 ** -(np.arange(0, rot, 2) / rot)
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


class Server:
    """A PagedCache driven like a scheduler does, next to its oracle."""

    def __init__(self, n_seq, hkv, dt, sink, recent, page, max_len, seed=0, rot=128, interleaved=False):
        from innerq_b200.paged import PagedCache
        self.r = np.random.RandomState(seed)
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.dt, self.hkv = DT[dt], hkv
        cols = max(1, -(-max_len // page))
        self.cache = PagedCache.allocate(n_seq * cols + 2, hkv, n_seq + 2, page, sink, recent, self.dt)
        self.cache.pages.fill_(0x5A)
        for d in (self.cache.dense_k, self.cache.dense_v):
            d.fill_(float("nan"))  # what was never written must never be seen
        self.table = torch.from_numpy(self.r.permutation(n_seq * cols + 2)[:n_seq * cols].reshape(n_seq, cols)
                                      .astype(np.int32)).cuda()
        self.slots = torch.from_numpy(self.r.permutation(n_seq + 2)[:n_seq].astype(np.int32)).cuda()
        self.lens = np.zeros(n_seq, np.int32)
        self.oracle = Oracle(sink, recent, self.dt)
        self.rot, self.interleaved = rot, interleaved
        self.cos, self.sin = table(max_len + 1, rot) if rot else (None, None)
        self.size = torch.exp(torch.randn((hkv, D), device="cuda", generator=self.g))

    def dev(self, x):
        return torch.from_numpy(np.asarray(x, np.int32)).cuda()

    def step(self, new, hq=0, seqs=None, one=False, kv=None):
        """Append new[i] tokens to sequence seqs[i]; returns (got q, expected q)."""
        seqs = np.arange(len(new)) if seqs is None else np.asarray(seqs)
        T = int(np.sum(new))
        x = torch.randn((T, hq + 2 * self.hkv, D), device="cuda", generator=self.g)
        x[:, hq:hq + self.hkv] *= self.size
        x = x.to(self.dt)
        if kv is not None:
            kv(x[:, hq:hq + self.hkv], x[:, hq + self.hkv:])
        at = torch.from_numpy(seqs).cuda()
        cs = dict(cos=torch.from_numpy(self.cos).cuda(), sin=torch.from_numpy(self.sin).cuda(),
                  interleaved=self.interleaved) if self.rot else {}
        q, k = self.cache.append(x[:, :hq] if hq else None, x[:, hq:hq + self.hkv], x[:, hq + self.hkv:], self.table[at],
                                 self.slots[at], self.dev(self.lens[seqs]),
                                 None if one else self.dev(np.concatenate([[0], np.cumsum(new)])), return_k=True, **cs)
        n = x.float().cpu().numpy()
        pos = np.concatenate([self.lens[b] + np.arange(c) for b, c in zip(seqs, new)] + [np.zeros(0, np.int64)]).astype(int)
        turn = lambda y: self.oracle.rnd(rotate64(y, self.cos[pos], self.sin[pos], self.interleaved)) if self.rot else y  # noqa: E731
        wq, wk = turn(n[:, :hq]), turn(n[:, hq:hq + self.hkv])
        o = 0
        for b, c in zip(seqs, new):
            self.oracle.append(b, wk[o:o + c], n[o:o + c, hq + self.hkv:])
            self.lens[b] += c
            o += c
        np.testing.assert_array_equal(k.float().cpu().numpy(), wk)
        if hq:
            np.testing.assert_array_equal(q.float().cpu().numpy(), wq)

    def check_read(self, seqs=None):
        """Every token of the sequences reads back as the oracle holds it, bit for bit."""
        seqs = np.arange(len(self.lens)) if seqs is None else np.asarray(seqs)
        n = self.lens[seqs]
        at = torch.from_numpy(seqs).cuda()
        k, v = self.cache.read(self.table[at], self.slots[at], self.dev(n), self.dev(np.zeros_like(n)),
                               self.dev(np.concatenate([[0], np.cumsum(n)])), int(n.sum()))
        o = 0
        for b, c in zip(seqs, n):
            if c:
                np.testing.assert_array_equal(k[o:o + c].float().cpu().numpy(), self.oracle.rnd(self.oracle.ck[b]))
                np.testing.assert_array_equal(v[o:o + c].float().cpu().numpy(), self.oracle.rnd(self.oracle.cv[b]))
            o += c

    def check_attend(self, hq, seqs=None, scale=None, dtype="fp16"):
        seqs = np.arange(len(self.lens)) if seqs is None else np.asarray(seqs)
        at = torch.from_numpy(seqs).cuda()
        q = torch.randn((len(seqs), hq, D), device="cuda", generator=self.g).to(self.dt)
        lse = torch.full((len(seqs), hq), 7.0, device="cuda")
        out = self.cache.attend(q, self.table[at], self.slots[at], self.dev(self.lens[seqs]), scale=scale, lse=lse)
        for i, b in enumerate(seqs):
            if b not in self.oracle.k:
                self.oracle.k[b] = self.oracle.v[b] = np.zeros((0, self.hkv, D), np.float32)
                self.oracle.ck[b] = self.oracle.cv[b] = np.zeros((0, self.hkv, D))
            want, wl = self.oracle.attend(b, q[i].float().cpu().numpy(), scale if scale is not None else D ** -0.5)
            close(out[i].double().cpu().numpy(), want, dtype, np.abs(np.nan_to_num(self.oracle.cv[b], nan=0, posinf=0, neginf=0)).max() if self.lens[b] else 1.0)
            np.testing.assert_allclose(lse[i].cpu().numpy(), wl, rtol=1e-5, atol=2e-3)


def close(got, want, dtype, vmax):
    """Each probability is rounded to 11 bits or more before it meets the
    values: an error of at most 2^-11 sum p |v| <= 2^-11 max |v|, and the
    output is rounded to its type."""
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    err = np.nan_to_num(np.abs(got - want))
    bound = ULP[dtype] * np.abs(np.nan_to_num(want)) + 2.0 ** -11 * vmax
    assert (err <= bound).all(), (err.max(), bound.flat[err.argmax()])


@pytest.mark.parametrize("dtype,hkv,hq,sink,recent,page,rot,inter", [
    ("fp16", 2, 8, 32, 96, 64, 128, False),
    ("bf16", 1, 5, 0, 0, 32, 64, False),
    ("fp16", 3, 3, 64, 32, 128, 128, True),
    ("bf16", 2, 14, 32, 0, 256, 32, True),
    ("fp16", 1, 8, 0, 32, 32, 0, False),
])
def test_prompts_then_decode(dtype, hkv, hq, sink, recent, page, rot, inter):
    """Ragged prompts (one of no tokens, one of one), chunks of them, then
    single tokens across several flushes; everything read back bit for bit and
    attended to."""
    s = Server(5, hkv, dtype, sink, recent, page, 700, seed=hq, rot=rot, interleaved=inter)
    s.step([1, 0, 33, 257, 128], hq)
    s.check_read()
    s.step([70, 5, 64, 130, 31], hq)  # chunks that begin anywhere
    s.check_read()
    s.check_attend(hq, dtype=dtype)
    for i in range(70):
        s.step([1] * 5, hq, one=True)
        if i % 23 == 0:
            s.check_read()
    s.check_read()
    s.check_attend(hq, dtype=dtype)


@pytest.mark.parametrize("length", [0, 1, 2, 31, 32, 33, 63, 64, 65, 95, 96, 97, 127, 128, 129, 160, 161, 191, 192, 193, 1000])
def test_every_length_near_the_seams(length):
    s = Server(2, 1, "fp16", 32, 32, 64, 1100, seed=length)
    s.step([length, 5], 4)
    s.check_read()
    s.check_attend(4)


@pytest.mark.parametrize("ratio", [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_head_ratios(ratio, dtype):
    s = Server(3, 2, dtype, 32, 32, 32, 900, seed=ratio)
    s.step([300, 801, 40], 2 * ratio)
    s.check_attend(2 * ratio, dtype=dtype)


def test_subset_order_and_scale():
    """Rows of a batch are any sequences in any order, one of them unused."""
    s = Server(6, 2, "fp16", 32, 96, 64, 3000, seed=3)
    s.step([2500, 10, 600, 0, 77, 1203], 8)
    s.check_attend(8, seqs=[5, 0, 3, 2])
    s.check_attend(8, seqs=[4], scale=0.3)
    s.check_attend(8, seqs=[0, 1], scale=0.0)
    s.check_attend(8, seqs=[0, 1], scale=-0.1)


def test_long_and_many():
    """Work split over many blocks, and many short sequences."""
    s = Server(1, 1, "fp16", 32, 96, 128, 40000, seed=4)
    s.step([39001], 4)
    s.check_attend(4)
    n = np.random.RandomState(5).randint(0, 150, 300)
    s = Server(300, 1, "bf16", 0, 32, 32, 160, seed=5)
    s.step(n, 2)
    s.check_attend(2, dtype="bf16")


def test_values_that_are_not_finite_stay_in_their_groups():
    """A NaN or an infinity in a quantized group makes that group NaN (key:
    32 channels of a token; value: one channel of 32 tokens) and nothing else;
    the attention is NaN exactly where the formula says."""
    s = Server(2, 1, "fp16", 0, 0, 32, 400, seed=6, rot=0)

    def poison(k, v):
        v[40, 0, 7] = float("inf")
        v[100, 0, 9] = float("nan")
    s.step([200, 90], 2, kv=poison)
    s.check_read()
    s.check_attend(2)

    def poison_key(k, v):
        k[5, 0, 70] = float("-inf")
    s.step([64, 64], 2, kv=poison_key)
    s.check_read()
    s.check_attend(2, seqs=[1])


def test_zero_groups_and_extremes():
    """Groups of zeros, of the type's smallest and largest values."""
    s = Server(1, 1, "fp16", 0, 0, 32, 200, seed=7, rot=0)

    def edge(k, v):
        k[:32] = 0
        v[32:64] = 0
        k[64:96] *= 2.0 ** -24 / k[64:96].abs().clamp(min=2.0 ** -24)
        v[96:128, 0, :5] = 65504.0
    s.step([160], 2, kv=edge)
    s.check_read()


def test_strided_inputs_and_streams():
    """Slices of a fused projection with an odd width, work on a stream of its
    own, outputs into a strided view."""
    from innerq_b200.paged import PagedCache
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn((3, 4 + 2 + 2 + 1, 136), device="cuda", generator=g).half()
    args = dict(page_table=torch.zeros((3, 1), dtype=torch.int32, device="cuda"),
                slots=torch.arange(3, dtype=torch.int32, device="cuda"))
    zero = torch.zeros(3, dtype=torch.int32, device="cuda")
    outs = []
    for contiguous in (False, True):
        c = PagedCache.allocate(1, 2, 3, 32, 0, 32)
        y = x[..., 3:131]  # rows that begin inside a 16-byte word
        q, k, v = y[:, :4], y[:, 4:6], y[:, 6:8]
        if contiguous:
            q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            qr = c.append(q, k, v, seq_lens=zero, **args)
            wide = torch.zeros((3, 4, 256), dtype=torch.float16, device="cuda")
            out = c.attend(qr, seq_lens=zero + 1, out=wide[..., 64:192], **args)
        torch.cuda.current_stream().wait_stream(st)
        assert torch.equal(qr, q) and (wide[..., :64] == 0).all() and (wide[..., 192:] == 0).all()
        outs.append(out.clone())
        want = v.repeat_interleave(2, 1)  # one token: its value
        assert torch.equal(out, want)
    assert torch.equal(*outs)


def test_names_out_of_range_are_nan_and_write_nothing():
    """A page, slot or position that does not exist: NaN, nothing written."""
    from innerq_b200.paged import PagedCache
    c = PagedCache.allocate(2, 1, 1, 32, 0, 0)
    c.pages.zero_(), c.dense_k.zero_(), c.dense_v.zero_()
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn((70, 4, 128), device="cuda", generator=g).half()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for tab, slot in ((i32(0, 1), 3), (i32(7, -1), 0)):
        c.append(x[:, :2], x[:, 2:3], x[:, 3:], tab[None], i32(slot), i32(0), i32(0, 70))
        if slot:
            assert int(c.pages.count_nonzero()) == 0 and int(c.dense_k.count_nonzero()) == 0
        assert torch.isnan(c.attend(x[:1, :2], tab[None], i32(slot), i32(70))).all()
    # more tokens than the table has pages for
    assert torch.isnan(c.attend(x[:1, :2], i32(0)[None], i32(0), i32(100))).all()
    assert torch.equal(c.attend(x[:1, :2], i32(0)[None], i32(0), i32(-5)), torch.zeros_like(x[:1, :2]))
    cs = torch.ones((10, 64), device="cuda")
    q = c.append(x[:12, :2], x[:12, 2:3], x[:12, 3:], i32(0, 1)[None], i32(0), i32(0), i32(0, 12), cos=cs, sin=cs)
    assert torch.isnan(q[10:]).all() and not torch.isnan(q[:10]).any()
    k, v = c.read(i32(0, 1)[None], i32(0), i32(12), i32(-1), i32(0, 14), 14)
    bad = torch.isnan(k).all(-1)[:, 0]
    assert bad.tolist() == [True] + [False] * 10 + [True] * 3  # 10, 11: keys without an angle
    assert torch.isnan(v).all(-1)[:, 0].tolist() == [True] + [False] * 12 + [True]


def test_decode_step_in_a_graph():
    """Append and attend recorded once, replayed while the lengths move on the device."""
    s = Server(3, 2, "fp16", 32, 32, 64, 500, seed=10)
    s.step([100, 37, 250], 8)
    lens = s.dev(s.lens)
    x = torch.empty((3, 12, D), dtype=torch.float16, device="cuda")
    out = torch.empty((3, 8, D), dtype=torch.float16, device="cuda")
    cos, sin = torch.from_numpy(s.cos).cuda(), torch.from_numpy(s.sin).cuda()

    def one():
        q = s.cache.append(x[:, :8], x[:, 8:10], x[:, 10:], s.table, s.slots, lens, cos=cos, sin=sin)
        lens.add_(1)
        s.cache.attend(q, s.table, s.slots, lens, out=out)
    x.normal_()
    keep = [t.clone() for t in (s.cache.pages, s.cache.dense_k, s.cache.dense_v, lens)]
    one()  # warm-up, undone
    for a, b in zip((s.cache.pages, s.cache.dense_k, s.cache.dense_v, lens), keep):
        a.copy_(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one()
    for i in range(40):
        x.normal_()
        graph.replay()
        n = x.float().cpu().numpy()
        pos = s.lens.astype(int)
        rot = lambda y: s.oracle.rnd(rotate64(y, s.cos[pos], s.sin[pos], False))  # noqa: E731
        q, k = rot(n[:, :8]), rot(n[:, 8:10])
        for b in range(3):
            s.oracle.append(b, k[b:b + 1], n[b:b + 1, 10:])
            s.lens[b] += 1
        if i % 13 == 0 or i == 39:
            for b in range(3):
                want, _ = s.oracle.attend(b, q[b], D ** -0.5)
                close(out[b].double().cpu().numpy(), want, "fp16", np.abs(s.oracle.cv[b]).max())
    s.check_read()


def test_refusals():
    """Arguments of the wrong shape, type or device raise before any launch."""
    from innerq_b200 import _lib
    from innerq_b200.paged import PagedCache
    from innerq_b200.prompt import prompt_attention
    c = PagedCache.allocate(4, 2, 2, 64, 32, 32)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    x = lambda n, h: torch.zeros((n, h, D), dtype=torch.float16, device="cuda")  # noqa: E731
    tab, sl, ln = i32(2, 3), i32(2), i32(2)
    with pytest.raises(ValueError):
        PagedCache(c.pages, c.dense_k, c.dense_v, 32, 64)  # another window than the slots have
    with pytest.raises(ValueError):
        PagedCache(c.pages, c.dense_k, c.dense_v, 16, 48)
    with pytest.raises(ValueError):
        PagedCache(c.pages[..., :4000], c.dense_k, c.dense_v, 32, 32)
    with pytest.raises(NotImplementedError):
        PagedCache(c.pages, c.dense_k[..., :64].contiguous(), c.dense_v[..., :64].contiguous(), 32, 32)
    with pytest.raises(TypeError):
        PagedCache(c.pages, c.dense_k.float(), c.dense_v.float(), 32, 32)
    with pytest.raises(ValueError):
        PagedCache.allocate(4, 2, 2, 48)
    with pytest.raises(TypeError):
        c.attend(x(2, 4), tab.long(), sl, ln)
    with pytest.raises(TypeError):
        c.attend(x(2, 4), tab, sl, ln.cpu())
    with pytest.raises(ValueError):
        c.attend(x(2, 4), tab, sl[:1], ln)
    with pytest.raises(ValueError):
        c.attend(x(3, 4), tab, sl, ln)
    with pytest.raises(TypeError):
        c.attend(x(2, 4).bfloat16(), tab, sl, ln)
    with pytest.raises(_lib.InnerqError):
        c.attend(x(2, 5), tab, sl, ln)  # not a multiple of the key heads
    with pytest.raises(_lib.InnerqError):
        c.attend(x(2, 18), tab, sl, ln)  # more than eight query heads to a key head
    with pytest.raises(ValueError):
        c.attend(x(2, 4), tab, sl, ln, out=x(2, 6))
    with pytest.raises(ValueError):
        c.attend(x(2, 4), tab, sl, ln, lse=torch.zeros((2, 5), device="cuda"))
    with pytest.raises(ValueError):
        c.append(None, x(3, 2), x(3, 2), tab, sl, ln)  # three tokens, two sequences, no cu_seqlens
    with pytest.raises(ValueError):
        c.append(None, x(2, 3), x(2, 3), tab, sl, ln)
    with pytest.raises(ValueError):
        c.append(x(1, 4), x(2, 2), x(2, 2), tab, sl, ln)
    with pytest.raises(ValueError):
        c.append(None, x(2, 2), x(2, 2), tab, sl, ln, cos=torch.zeros((4, 64), device="cuda"))
    with pytest.raises(TypeError):
        c.append(None, x(2, 2), x(2, 2), tab, sl, ln, cos=torch.zeros((4, 64), device="cuda").half(),
                 sin=torch.zeros((4, 64), device="cuda").half())
    with pytest.raises(_lib.InnerqError):
        c.append(None, x(2, 2), x(2, 2), tab, sl, ln, cos=torch.zeros((4, 12), device="cuda"), sin=torch.zeros((4, 12), device="cuda"))
    q, k = x(4, 4), x(4, 2)
    with pytest.raises(ValueError):
        prompt_attention(q, k, x(5, 2), i32(2))
    with pytest.raises(TypeError):
        prompt_attention(q, k.bfloat16(), k, i32(2))
    with pytest.raises(ValueError):
        prompt_attention(q, k, k, i32(2), i32(3))
    with pytest.raises(TypeError):
        prompt_attention(q, k, k, i32(2).long())
    with pytest.raises(_lib.InnerqError):
        prompt_attention(x(4, 3), k, k, i32(2))
    with pytest.raises(TypeError):
        prompt_attention(q.float(), k.float(), k.float(), i32(2))


def test_nothing_to_do():
    """No sequences, no tokens."""
    from innerq_b200.paged import PagedCache
    from innerq_b200.prompt import prompt_attention
    c = PagedCache.allocate(1, 2, 1, 32, 0, 0)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    x = lambda n, h: torch.zeros((n, h, D), dtype=torch.float16, device="cuda")  # noqa: E731
    assert c.attend(x(0, 4), i32(0, 1), i32(0), i32(0)).shape == (0, 4, D)
    assert c.append(x(0, 4), x(0, 2), x(0, 2), i32(0, 1), i32(0), i32(0)).shape == (0, 4, D)
    k, v = c.read(i32(0, 1), i32(0), i32(0), i32(0), i32(1), 0)
    assert k.shape == v.shape == (0, 2, D)
    assert prompt_attention(x(0, 4), x(0, 2), x(0, 2), i32(1)).shape == (0, 4, D)
    # queries without any keys in the whole call
    cu = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    assert torch.equal(prompt_attention(x(3, 4) + 1, x(0, 2), x(0, 2), cu, i32(2)), x(3, 4))
    # a sequence whose page table has no columns: only the 16-bit rows count
    kv = torch.ones((1, 2, D), dtype=torch.float16, device="cuda")
    c.append(None, kv, kv, i32(1, 0), i32(1), i32(1))
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    assert torch.equal(c.attend(x(1, 4), i32(1, 0), i32(1), one), x(1, 4) + 1)


@pytest.mark.parametrize("dtype,hq", [("fp16", 8), ("fp16", 5), ("bf16", 8)])
def test_long_contexts_have_no_error_of_one_sign(dtype, hq):
    """What a tile's sums lose must not add up over a long context.  Errors of
    one sign show along the values' sizes: there the rounding of the output and
    of the probabilities (each at most 2^-11 / sqrt 3 rms for fp16; the
    output's is 2^-8 / sqrt 3 for bf16) leaves about 1 / sqrt 128 of itself per
    row.  The limit is four such deviations of the rows' mean, and 1e-4 for
    what the sums may lose."""
    s = Server(2, 2, dtype, 32, 96, 128, 33000, seed=21)
    s.step([33000, 21003])
    rows = []
    at = torch.arange(2).cuda()
    q = torch.randn((2, 2 * hq, D), device="cuda", generator=s.g).to(s.dt)
    out = s.cache.attend(q, s.table[at], s.slots[at], s.dev(s.lens)).double().cpu().numpy()
    for b in range(2):
        want, _ = s.oracle.attend(b, q[b].float().cpu().numpy(), D ** -0.5)
        for h in range(2 * hq):
            size = np.abs(s.oracle.cv[b][:, h // hq]).mean(0)
            rows.append((out[b, h] - want[h]) @ size / np.linalg.norm(size) / np.linalg.norm(want[h]))
    deviation = math.hypot(ULP[dtype], 2.0 ** -11) / math.sqrt(3 * D)
    assert abs(np.mean(rows)) < 4 * deviation / math.sqrt(len(rows)) + 1e-4, (np.mean(rows), np.max(np.abs(rows)))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("rot", [0, 64, 128])
@pytest.mark.parametrize("one", [True, False])
def test_tokens_of_no_sequence_are_nan_and_write_nothing(one, rot, dtype):
    """A negative length (a padding row of a batch) and tokens past the last
    sequence: NaN in every channel of the rotated queries and keys, nothing
    written, the other tokens as without them."""
    from innerq_b200.paged import PagedCache
    g = torch.Generator(device="cuda").manual_seed(22)
    n = 3 if one else 40
    x = torch.randn((n, 5 + 2 + 2, D), device="cuda", generator=g).to(DT[dtype])
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    cos, sin = (torch.from_numpy(t).cuda() for t in table(64, rot)) if rot else (None, None)
    tab = i32(0, 1, 2)[:, None]
    results = []
    for lens, cu in ((i32(4, -1, 2), [0, 9, 20, 31]), (i32(4, 0, 2), [0, 9, 20, 40])):
        c = PagedCache.allocate(3, 2, 3, 32, 32, 32, DT[dtype])
        c.pages.fill_(1), c.dense_k.fill_(1), c.dense_v.fill_(1)
        old = [torch.full((n, h, D), 7.0, dtype=DT[dtype], device="cuda") for h in (5, 2, 5, 2)]
        del old  # what the allocator hands out next
        q, k = c.append(x[:, :5], x[:, 5:7], x[:, 7:], tab, i32(0, 1, 2), lens, None if one else i32(*cu), cos=cos, sin=sin,
                        return_k=True)
        results.append((q, k, c))
    (q, k, c), (q1, k1, c1) = results
    lost = torch.zeros(n, dtype=torch.bool, device="cuda")
    lost[1:2] = one
    if not one:
        lost[9:20] = lost[31:] = True
    for got, whole in ((q, q1), (k, k1)):
        assert torch.isnan(got[lost]).all()
        assert torch.equal(got[~lost], whole[~lost])
    assert (c.dense_k[1] == 1).all() and (c.dense_v[1] == 1).all() and (c.pages == 1).all()
    assert torch.equal(c.dense_k[0], c1.dense_k[0])
    if not one:  # no sequences at all
        q, k = c.append(x[:, :5], x[:, 5:7], x[:, 7:], tab[:0], i32(), i32(), i32(0), cos=cos, sin=sin, return_k=True)
        assert torch.isnan(q).all() and torch.isnan(k).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("length", [20, 90, 700, 9000])
def test_infinite_values_of_the_16_bit_tokens(length, dtype):
    """An infinity in the sink or the window, times any probability above 0, is
    an infinity: of its sign, in its channel, in every query's output.  Two of
    both signs, or a NaN, are NaN.  The other channels do not change by a bit.
    One of the infinities sits at a token whose probability is below what fp16
    holds."""
    from innerq_b200.paged import PagedCache
    g = torch.Generator(device="cuda").manual_seed(length)
    x = torch.randn((length, 2, D), device="cuda", generator=g).to(DT[dtype])
    q = torch.randn((1, 8, D), device="cuda", generator=g).to(DT[dtype])
    q[..., 0] = 8.0
    x[:, 0, 0] = 0
    x[7, 0, 0] = -40.0  # logit 8 * -40 / sqrt 128 = -28: 2^-41
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    tab = torch.arange(-(-length // 64), dtype=torch.int32, device="cuda")[None]
    last = length - 1
    inf, nan = float("inf"), float("nan")
    outs = []
    for bad in (False, True):
        v = x[:, 1:].clone()
        for t, d, y in ((3, 10, inf), (4, 11, -inf), (last, 12, inf), (last - 2, 13, -inf), (3, 14, inf), (last, 14, -inf),
                        (last - 5, 15, nan), (7, 16, inf), (7, 17, -inf)):
            v[t, 0, d] = y if bad else 0.0
        c = PagedCache.allocate(tab.shape[1], 1, 1, 64, 32, 32, DT[dtype])
        c.append(None, x[:, :1], v, tab, i32(0), i32(0), i32(0, length))
        outs.append(c.attend(q, tab, i32(0), i32(length))[0].double().cpu())
    clean, got = outs
    want = {10: inf, 11: -inf, 12: inf, 13: -inf, 14: nan, 15: nan, 16: inf, 17: -inf}
    for d, w in want.items():
        assert torch.equal(got[:, d], torch.full((8,), w, dtype=torch.float64)) or (w != w and torch.isnan(got[:, d]).all()), (d, got[:, d])
    keep = [d for d in range(D) if d not in want]
    assert torch.equal(got[:, keep], clean[:, keep])


def held(c, pages, length, slot=0):
    """What a cache holds of a sequence, [length, H, D] in 64 bits."""
    t, d = torch.arange(32, device="cuda")[:, None], torch.arange(D, device="cuda")[None]
    H, dt, sink = c.n_kv_heads, c.dtype, c.w_sink
    n = c.packed_tokens(length)
    blocks = c.pages[pages.long()].transpose(0, 1).reshape(H, -1, 4608)[:, :n // 32]
    scale = lambda lo: blocks[..., lo:lo + 256].contiguous().view(dt).double()  # noqa: E731

    def code(base, word, nibble):
        return (blocks.long()[..., base + word * 4 + nibble // 2] >> (4 * (nibble % 2))) % 16 - 8
    g, l, m = d // 32, d // 8 % 4, d % 8
    k = code(0, ((t // 8 * 8 + t % 8) * 4 + l) * 4 + g, m) * scale(2048)[..., (t % 8 * 4 + t // 8) * 4 + g]
    word = (((d // 4 % 4 * 8 + d // 16) * 4 + t % 8 // 2) * 2 + d // 2 % 2) * 2 + d % 2
    v = code(2304, word, t // 8 + 4 * (t % 2)) * scale(4352)[..., None, :]
    at = torch.cat([torch.arange(min(sink, length)), torch.arange(min(sink + n, length), length)]).cuda()
    row = torch.where(at < sink, at, sink + (at - sink) % (c.w_recent + 32))
    out = []
    for packed, dense in ((k, c.dense_k), (v, c.dense_v)):
        x = torch.empty((length, H, D), dtype=torch.float64, device="cuda")
        if n:
            x[sink:sink + n] = packed.reshape(H, n, D).transpose(0, 1)
        x[at] = dense[slot][:, row].transpose(0, 1).double()
        out.append(x)
    return out


@pytest.mark.parametrize("kind", ["normal", "one sign", "outliers", "constant"])
@pytest.mark.parametrize("dtype,length,hq", [("fp16", 33000, 8), ("fp16", 120001, 8), ("bf16", 33000, 4)])
def test_sums_over_long_contexts_do_not_depend_on_how_codes_are_spread(dtype, length, hq, kind):
    """Values whose codes are spread, of one sign, nearly all zero (one large
    value per group) or all alike, against 64 bits over what the cache holds.
    Rounding of the output (2^-11 / sqrt 3 of a value in fp16, 2^-8 / sqrt 3 in
    bf16, at most) and of the probabilities to 11 bits (a random walk, 2^-11 /
    sqrt 3 of sqrt(sum p^2 v^2) at most) are all that may be left: the errors'
    mean along the values' sizes within four of its deviations, and a row's
    error within 1.25 of them together, the 128 channels' own scatter (four
    deviations of a root of a mean of 128 squares) included.  5e-5 for the sums
    in 32 bits."""
    from innerq_b200.paged import PagedCache
    dt, H = DT[dtype], 2
    g = torch.Generator(device="cuda").manual_seed(24)
    z = torch.randn((length, H, D), device="cuda", generator=g)
    if kind == "one sign":
        z = z.abs()
    elif kind == "constant":
        z = torch.full_like(z, 0.75)
    elif kind == "outliers":
        at = torch.randint(0, 32, (length // 32 + 1, 1, H, D), device="cuda", generator=g)
        big = (torch.arange(32, device="cuda")[None, :, None, None] == at).flatten(0, 1)[:length]
        z = torch.where(big, 20.0 * torch.sign(z), 0.5 * z)
    k = torch.randn((length, H, D), device="cuda", generator=g).to(dt)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    tab = torch.arange(length // 128 + 1, dtype=torch.int32, device="cuda")[None]
    c = PagedCache.allocate(tab.shape[1], H, 1, 128, 32, 96, dt)
    c.append(None, k, z.to(dt), tab, i32(0), i32(0), i32(0, length))
    q = torch.randn((1, H * hq, D), device="cuda", generator=g).to(dt)
    lse = torch.empty((1, H * hq), device="cuda")
    out = c.attend(q, tab, i32(0), i32(length), lse=lse)[0].double()
    kk, vv = held(c, tab[0], length)
    along, size_of_rounding = [], []
    for h in range(H):
        s = q[0, h * hq:h * hq + hq].double() @ kk[:, h].T * D ** -0.5
        p = torch.softmax(s, -1)
        want = p @ vv[:, h]
        err = out[h * hq:h * hq + hq] - want
        assert float((lse[0, h * hq:h * hq + hq].double() - torch.logsumexp(s, -1) / math.log(2)).abs().max()) < 1e-4
        walk = (p.square() @ vv[:, h].square()).sqrt()
        expect = ((ULP[dtype] * want).square() + (2.0 ** -11 * walk).square()).sum(-1).div(3 * D).sqrt()  # rms of a channel
        size = want.norm(dim=1) / D ** 0.5
        assert bool((err.norm(dim=1) / D ** 0.5 <= 1.25 * expect + 5e-5 * size).all()), (err.norm(dim=1) / D ** 0.5 / expect)
        if kind in ("normal", "outliers"):  # elsewhere the output's own rounding has a sign
            scale = vv[:, h].abs().mean(0)
            along += ((err @ scale) / scale.norm() / D ** 0.5 / size).tolist()
            size_of_rounding += (expect / size / D ** 0.5).tolist()
    if along:
        n = len(along)
        assert abs(sum(along) / n) <= 4 * sum(size_of_rounding) / n / n ** 0.5 + 5e-5, (sum(along) / n, sum(size_of_rounding) / n)


def test_launches_are_counted_where_kernels_are_launched():
    """Calls that are refused or have nothing to do count no launches."""
    from innerq_b200 import _lib
    from innerq_b200.paged import PagedCache
    from innerq_b200.prompt import prompt_attention
    c = PagedCache.allocate(4, 2, 2, 64, 32, 32)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    x = lambda n, h: torch.zeros((n, h, D), dtype=torch.float16, device="cuda")  # noqa: E731
    tab, sl, ln = i32(2, 3), i32(2), i32(2)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")

    def count(call, error=None):
        n = _lib.launch_count[0]
        if error:
            with pytest.raises(error):
                call()
        else:
            call()
        return _lib.launch_count[0] - n
    assert count(lambda: c.attend(x(3, 4), tab, sl, ln), ValueError) == 0
    assert count(lambda: c.attend(x(2, 5), tab, sl, ln), _lib.InnerqError) == 0
    assert count(lambda: c.append(None, x(3, 2), x(3, 2), tab, sl, ln), ValueError) == 0
    assert count(lambda: c.read(tab, sl, ln, ln, ln, 2), ValueError) == 0
    assert count(lambda: prompt_attention(x(4, 3), x(4, 2), x(4, 2), cu), _lib.InnerqError) == 0
    assert count(lambda: c.attend(x(0, 4), tab[:0], sl[:0], ln[:0])) == 0
    assert count(lambda: c.append(None, x(0, 2), x(0, 2), tab, sl, ln, i32(3))) == 0
    assert count(lambda: c.read(tab, sl, ln, ln, i32(3), 0)) == 0
    assert count(lambda: prompt_attention(x(0, 4), x(0, 2), x(0, 2), cu)) == 0
    assert count(lambda: c.append(None, x(2, 2), x(2, 2), tab, sl, ln)) == 1
    assert count(lambda: c.append(None, x(2, 2), x(2, 2), tab, sl, ln, cu)) == 2
    assert count(lambda: c.attend(x(2, 4), tab, sl, ln)) == 2
    assert count(lambda: c.read(tab, sl, ln, ln, cu, 2)) == 1
    assert count(lambda: prompt_attention(x(2, 4), x(2, 2), x(2, 2), cu)) == 1


def test_switches_without_a_truth_value_raise():
    """What has no truth value raises its own error, before any launch."""
    from innerq_b200.paged import PagedCache
    from innerq_b200.prompt import prompt_attention
    c = PagedCache.allocate(1, 1, 1, 32, 0, 32)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    x = torch.zeros((1, 1, D), dtype=torch.float16, device="cuda")
    cs = torch.ones((4, 64), device="cuda")
    many = torch.ones(2)
    c.dense_k.fill_(5)
    with pytest.raises(RuntimeError, match="ambiguous"):
        c.append(x, x, x, i32(0)[None], i32(0), i32(0), cos=cs, sin=cs, interleaved=many)
    with pytest.raises(RuntimeError, match="ambiguous"):
        c.append(x, x, x, i32(0)[None], i32(0), i32(0), return_k=many)
    with pytest.raises(RuntimeError, match="ambiguous"):
        prompt_attention(x, x, x, i32(0, 1), causal=many)
    assert (c.dense_k == 5).all()


@pytest.mark.parametrize("dtype,page,sink,recent,longest", [("fp16", 64, 32, 96, 20000), ("bf16", 128, 0, 32, 60000),
                                                           ("fp16", 32, 0, 0, 3000)])
def test_every_tile_of_a_ragged_batch_counts_once(dtype, page, sink, recent, longest):
    """Bounds that shrink with the context, so that a tile missed, taken twice
    or weighted wrongly where the work is cut shows: it changes lse by 32 / n
    and the output by far more than its own size allows.  An element's error is
    at most the output's rounding and 2^-11 of sum p |v| and of the output (the
    probabilities' rounding, above and below the line).  Where at least 100
    tokens share the weight, the rounding of the probabilities is a random walk
    of steps of at most 2^-11 / sqrt 3 of p v, and a row's root mean square stays
    within 1.25 of both together.  The log-sum-exp is off by at most 2^-11 log2 e
    (the sum of the rounded probabilities), and by a walk of a tenth of that,
    below 1e-4, where 100 tokens share the weight."""
    from innerq_b200.paged import PagedCache
    dt, H, R = DT[dtype], 2, 3
    g = torch.Generator(device="cuda").manual_seed(26)
    r = np.random.RandomState(26)
    lens = np.concatenate([[1, 31, 33, longest], np.exp(r.uniform(0, np.log(longest), 20)).astype(int)])
    r.shuffle(lens)
    B, cols = len(lens), longest // page + 1
    tab = torch.from_numpy(r.permutation(B * cols).reshape(B, cols).astype(np.int32)).cuda()
    slots = torch.from_numpy(r.permutation(B).astype(np.int32)).cuda()
    c = PagedCache.allocate(B * cols, H, B, page, sink, recent, dt)
    T = int(lens.sum())
    i32 = lambda x: torch.from_numpy(np.asarray(x, np.int32)).cuda()  # noqa: E731
    k, v = (torch.randn((T, H, D), device="cuda", generator=g).to(dt) for _ in range(2))
    c.append(None, k, v, tab, slots, i32(np.zeros(B)), i32(np.concatenate([[0], np.cumsum(lens)])))
    q = (torch.randn((B, H * R, D), device="cuda", generator=g) * torch.tensor([0.0, 0.3, 1.0] * H, device="cuda")[:, None]).to(dt)
    lse = torch.empty((B, H * R), device="cuda")
    out = c.attend(q, tab, slots, i32(lens), lse=lse).double()
    for b, n in enumerate(lens):
        kk, vv = held(c, tab[b], int(n), int(slots[b]))
        for h in range(H):
            rows = slice(h * R, h * R + R)
            s = q[b, rows].double() @ kk[:, h].T * D ** -0.5
            p = torch.softmax(s, -1)
            want = p @ vv[:, h]
            err = (out[b, rows] - want).abs()
            many = p.square().sum(-1) < 0.01
            off = (lse[b, rows].double() - torch.logsumexp(s, -1) / math.log(2)).abs()
            assert bool((off < torch.where(many, 1e-4, 2.0 ** -11 * math.log2(math.e) + 1e-5)).all()), (b, n, off)
            assert bool((err <= ULP[dtype] * want.abs() + 2.0 ** -11 * (p @ vv[:, h].abs() + want.abs()) + 1e-6).all()), (b, n)
            walk = (p.square() @ vv[:, h].square()).sqrt()
            expect = ((ULP[dtype] * want).square() + (2.0 ** -11 * walk).square()).mean(-1).div(3).sqrt()
            assert bool((err.square().mean(-1).sqrt() <= 1.25 * expect + 1e-6)[many].all()), (b, n)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_same_inputs_same_bits(dtype):
    """Append, read-back and attention repeat themselves bit for bit, whatever
    ran between."""
    s = Server(7, 2, dtype, 32, 96, 64, 9000, seed=29)
    s.step([8500, 1, 77, 3000, 129, 640, 33], 10)
    q = torch.randn((7, 10, D), device="cuda", generator=s.g).to(s.dt)
    lens = s.dev(s.lens)
    first = s.cache.attend(q, s.table, s.slots, lens)
    other = Server(3, 1, dtype, 0, 32, 32, 4000, seed=30)
    for fill in (1e4, float("nan"), 0.0):
        def values(k, v):
            k[:], v[:] = fill, fill
        other.lens[:] = 0
        other.oracle = Oracle(0, 32, other.dt)
        other.rot = 0
        other.step([3000, 50, 1], kv=values)
        other.cache.attend(torch.full((3, 8, D), fill, dtype=other.dt, device="cuda"), other.table, other.slots, other.dev(other.lens))
        assert torch.equal(s.cache.attend(q, s.table, s.slots, lens), first)
    s.check_read()
