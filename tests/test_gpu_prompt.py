"""Attention over packed prompts against the formula in 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
ULP = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}


def cu(n):
    return torch.from_numpy(np.concatenate([[0], np.cumsum(n)]).astype(np.int32)).cuda()


def reference(q, k, v, nq, nk, causal, scale):
    """out [Tq, Hq, D], lse [Tq, Hq] (base 2), the largest |v| a row can see [Tq, Hq], in float64."""
    q, k, v = q.double(), k.double(), v.double()
    R = q.shape[1] // k.shape[1]
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], float("-inf"), dtype=torch.float64, device=q.device)
    vmax = torch.zeros_like(lse)
    o = p = 0
    for a, b in zip(nq, nk):
        if a and b:
            kk, vv = (x[p:p + b].repeat_interleave(R, 1).transpose(0, 1) for x in (k, v))
            i, j = torch.arange(a, device=q.device)[:, None], torch.arange(b, device=q.device)
            seen = (j <= i + b - a) if causal else torch.ones((a, b), dtype=torch.bool, device=q.device)
            s = (q[o:o + a].transpose(0, 1) @ kk.transpose(1, 2)) * scale
            s = torch.where(seen, s, float("-inf"))  # whatever is there
            m = s.amax(-1, keepdim=True)
            e = torch.where(seen & (m > float("-inf")), torch.exp(s - m), torch.where(torch.isnan(m) & seen, m, 0.0))
            l = e.sum(-1, keepdim=True)
            w = torch.where(l == 0, 0.0, e / torch.where(l == 0, 1.0, l))
            for r0 in range(0, a, 256):  # a masked value does not count, a seen one does even with weight 0
                ww, ss = w[:, r0:r0 + 256], seen[r0:r0 + 256]
                bad = ~torch.isfinite(vv)
                res = ww @ torch.where(bad, 0.0, vv)
                if bad.any():
                    hit = ss.double() @ bad.double()
                    for h in range(q.shape[1]):
                        for r, d in zip(*torch.nonzero(hit[h], as_tuple=True)):
                            res[h, r, d] = (ww[h, r, ss[r]] * vv[h, ss[r], d]).sum()
                out[o + r0:o + min(a, r0 + 256)] = res.transpose(0, 1)
            lse[o:o + a] = ((m + torch.log(l)) / np.log(2.0))[..., 0].T
            vmax[o:o + a] = torch.nan_to_num(vv, 0, 0, 0).abs().amax((1, 2))[None].expand(a, -1)
        o, p = o + a, p + b
    return out, lse, vmax


def check(q, k, v, nq, nk, causal, dtype, scale=None, **kw):
    from innerq_b200.prompt import prompt_attention
    lse = torch.full(q.shape[:2], 3.0, device="cuda")
    out = prompt_attention(q, k, v, cu(nq), None if nk is nq else cu(nk), scale=scale, causal=causal, lse=lse, **kw)
    want, wl, vmax = reference(q, k, v, nq, nk, causal, D ** -0.5 if scale is None else scale)
    n = int(sum(nq))
    got, want, wl, vmax = out[:n].double(), want[:n], wl[:n], vmax[:n]
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    # probabilities are rounded to the type before they meet the values, the
    # output is rounded to its type
    err = torch.nan_to_num(got - want).abs()
    bound = ULP[dtype] * (torch.nan_to_num(want).abs() + vmax[..., None])
    assert bool((err <= bound).all()), float((err - bound).max())
    fine = torch.isfinite(wl)
    assert torch.equal(torch.isneginf(lse[:n]), torch.isneginf(wl))
    assert bool(((lse[:n].double() - wl)[fine].abs() <= 2e-3 + 1e-5 * wl[fine].abs()).all())
    return out


def data(nq, nk, hq, hkv, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda n, h: torch.randn((int(sum(n)), h, D), device="cuda", generator=g).to(DT[dtype])  # noqa: E731
    return r(nq, hq), r(nk, hkv), r(nk, hkv)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n", [[1], [2, 1, 3], [127], [128], [129], [255, 1, 257], [0, 300, 0, 64, 1, 0], [513, 40], [1030]])
def test_lengths(n, causal, dtype):
    q, k, v = data(n, n, 4, 2, dtype, seed=sum(n))
    check(q, k, v, n, n, causal, dtype)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 3), (6, 2), (5, 1), (8, 8), (16, 2), (40, 8), (7, 1), (20, 1), (32, 1), (33, 1), (64, 1)])
def test_heads(hq, hkv):
    n = [200, 77]
    q, k, v = data(n, n, hq, hkv, "fp16", seed=hq)
    check(q, k, v, n, n, True, "fp16")


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("nq,nk", [([1], [1000]), ([1, 1, 1], [5, 300, 129]), ([64, 200], [1000, 200]), ([130, 5], [131, 900]),
                                   ([10, 300, 8], [4, 100, 0]), ([300], [1]), ([257, 0, 3], [130, 50, 3])])
def test_keys_longer_or_shorter_than_queries(nq, nk, causal):
    """A chunk sees what came before it; more queries than keys leave rows
    that see nothing: zeros."""
    q, k, v = data(nq, nk, 4, 2, "bf16", seed=sum(nq) + sum(nk))
    check(q, k, v, nq, nk, causal, "bf16")


def test_many_sequences():
    """More sequences than a warp, some empty; more pieces of work than CTAs."""
    r = np.random.RandomState(11)
    nq = np.where(r.rand(700) < 0.2, 0, r.randint(1, 40, 700)).tolist()
    q, k, v = data(nq, nq, 4, 2, "fp16", seed=12)
    check(q, k, v, nq, nq, True, "fp16")
    nk = [n + int(x) for n, x in zip(nq, r.randint(0, 200, 700))]
    q, k, v = data(nq, nk, 2, 2, "bf16", seed=13)
    check(q, k, v, nq, nk, True, "bf16")


def test_long():
    n = [5000, 1, 3001]
    q, k, v = data(n, n, 2, 1, "fp16", seed=1)
    check(q, k, v, n, n, True, "fp16")


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.05, 3e-3])
def test_scales(scale):
    """Peaked and flat distributions; logits far beyond the exponent's range."""
    n = [300, 170]
    q, k, v = data(n, n, 2, 2, "fp16", seed=2)
    check(q * 4, k, v, n, n, True, "fp16", scale=scale)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_masked_places_may_hold_anything(bad, dtype):
    """Values and keys that are not finite reach exactly the queries that see
    them: not earlier tokens, not the neighbouring sequences."""
    n = [200, 140, 300]
    q, k, v = data(n, n, 2, 1, dtype, seed=3)
    v[200 + 139] = bad  # the last token of the second sequence
    v[50, 0, 3] = bad
    check(q, k, v, n, n, True, dtype)
    q, k, v = data(n, n, 2, 1, dtype, seed=4)
    k[150] = float("nan")
    check(q, k, v, n, n, True, dtype)
    q, k, v = data(n, n, 2, 1, dtype, seed=5)
    k[199, 0] = float("nan")
    v[199, 0] = bad
    check(q, k, v, n, n, True, dtype)


def test_rising_logits():
    """A running maximum that grows from key to key by more than any
    deferred rescaling allows."""
    n = [700]
    q, k, v = data(n, n, 2, 1, "bf16", seed=6)
    q[:] = 1.0
    k[:] = (torch.arange(700, device="cuda") / 8.0)[:, None, None].to(torch.bfloat16)
    check(q, k, v, n, n, True, "bf16", scale=0.25)
    check(q, k, v, n, n, True, "bf16", scale=-0.25)


def test_rows_past_the_last_sequence_are_left_alone():
    n = [100, 60]
    q, k, v = data([200], [200], 2, 1, "fp16", seed=7)
    k[160:], v[160:] = float("nan"), float("nan")
    out = torch.full((200, 2, D), 5.0, dtype=torch.float16, device="cuda")
    check(q, k, v, n, n, True, "fp16", out=out)
    assert (out[160:] == 5).all()


def test_strides_and_streams():
    """q, k, v as slices of one projection; a stream of its own; out strided."""
    from innerq_b200.prompt import prompt_attention
    n = [130, 31]
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn((161, 8, 144), device="cuda", generator=g).half()
    for view in (x[..., :128], x[..., 8:136], x[..., 5:133]):
        q, k, v = view[:, :4], view[:, 4:6], view[:, 6:]
        wide = torch.zeros((161, 4, 256), dtype=torch.float16, device="cuda")
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            prompt_attention(q, k, v, cu(n), out=wide[..., 64:192])
        torch.cuda.current_stream().wait_stream(st)
        want = prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), cu(n))
        assert torch.equal(wide[..., 64:192], want)
        assert (wide[..., :64] == 0).all() and (wide[..., 192:] == 0).all()
    check(q.contiguous(), k.contiguous(), v.contiguous(), n, n, True, "fp16")


def test_same_inputs_same_bits():
    from innerq_b200.prompt import prompt_attention
    n = [1000, 333]
    q, k, v = data(n, n, 4, 2, "bf16", seed=9)
    a = prompt_attention(q, k, v, cu(n))
    assert torch.equal(a, prompt_attention(q, k, v, cu(n)))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("ratio", [2, 3, 5, 6, 7, 32, 33])
def test_bits_do_not_depend_on_what_ran_before(ratio, dtype):
    """Ratios that leave rows of a query tile without a query: whatever an
    earlier call left in shared memory, the same inputs give the same bits."""
    from innerq_b200.prompt import prompt_attention
    n = [300, 77, 129]
    q, k, v = data(n, n, ratio, 1, dtype, seed=ratio)
    outs = []
    for fill in (0.0, 1.0, 300.0, float("nan"), float("inf")):
        other = torch.full((4000, 8, D), fill, dtype=DT[dtype], device="cuda")
        prompt_attention(other, other[:, :4].contiguous(), other[:, :4].contiguous(), cu([4000]))
        outs.append(prompt_attention(q, k, v, cu(n)))
    for o in outs[1:]:
        assert torch.equal(o, outs[0])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("hq,hkv", [(4, 2), (5, 1)])
def test_bits_do_not_depend_on_the_neighbours(hq, hkv, dtype):
    """A sequence alone and beside others: the same bits, whatever they hold."""
    from innerq_b200.prompt import prompt_attention
    q, k, v = data([200], [200], hq, hkv, dtype, seed=20)
    alone = prompt_attention(q, k, v, cu([200]))
    for fill in (1.0, -60.0, 60000.0, float("nan"), float("inf")):
        x = [torch.cat([t, torch.full((300, t.shape[1], D), fill, dtype=t.dtype, device="cuda")]) for t in (q, k, v)]
        assert torch.equal(prompt_attention(*x, cu([200, 300]))[:200], alone), fill


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("nk", [1, 100, 128, 129, 256, 300])
def test_rows_whose_logits_are_all_minus_infinity(nk, causal, dtype):
    """Keys with an infinite channel: softmax is 0 / 0, NaN, for every row that
    sees a key, at every length; a row that sees none gets zeros.  The
    log-sum-exp is -inf for both."""
    from innerq_b200.prompt import prompt_attention
    nq = [nk, nk + 10]
    q, k, v = data(nq, [nk, nk], 2, 1, dtype, seed=nk)
    q = q.abs() + 1
    k[..., 5] = float("-inf")
    lse = torch.zeros(q.shape[:2], device="cuda")
    out = prompt_attention(q, k, v, cu(nq), cu([nk, nk]), causal=causal, lse=lse)
    blind = torch.zeros(len(q), dtype=torch.bool, device="cuda")
    blind[nk:nk + 10] = causal  # ten queries more than keys
    assert torch.isnan(out[~blind]).all()
    assert (out[blind] == 0).all()
    assert torch.isneginf(lse).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("n", [128, 300, 513])
def test_keys_of_minus_infinity_have_no_weight(n, dtype):
    """Some keys with an infinite channel, whole key tiles among them: the
    others' softmax, whatever finite values those keys have."""
    q, k, v = data([n], [n], 2, 1, dtype, seed=n)
    q = q.abs()
    q[..., 5] = 1.0
    gone = torch.arange(n, device="cuda") % 3 == 1
    gone[128:256] = True
    k[gone, 0, 5] = float("-inf")
    for causal in (False, True):
        out = check(q, k, v, [n], [n], causal, dtype)
        other = v.clone()
        other[gone] = 60000.0
        assert torch.equal(check(q, k, other, [n], [n], causal, dtype), out)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n", [40, 128, 300, 1000])
def test_infinite_values_with_small_probabilities(n, causal, dtype):
    """An infinity times any probability above 0 is an infinity, also where the
    probability is below what fp16 holds (2^-41 here), in a key tile that all
    queries see whole as in one that they do not; of both signs it is NaN.  The
    other channels do not change by a bit."""
    from innerq_b200.prompt import prompt_attention
    q, k, v = data([n], [n], 5, 1, dtype, seed=n)
    q[..., 0], k[..., 0] = 8.0, 0.0
    k[[7, n - 3], 0, 0] = -40.0  # logit 8 * -40 / sqrt 128 = -28
    outs = []
    for inf in (0.0, float("inf")):
        v[[7, 7, n - 3, 7, n - 3], 0, [16, 17, 18, 19, 19]] = torch.tensor([inf, -inf, inf, inf, -inf]).to(v)
        outs.append(prompt_attention(q, k, v, cu([n]), causal=causal).double())
    clean, got = outs
    sees = lambda t: torch.arange(n, device="cuda")[:, None].expand(n, 5) >= (t if causal else 0)  # noqa: E731
    inf = float("inf")
    for d, t, sign in ((16, 7, inf), (17, 7, -inf), (18, n - 3, inf)):
        assert torch.equal(got[..., d], torch.where(sees(t), sign, clean[..., d])), d
    assert torch.equal(torch.nan_to_num(got[..., 19], nan=7.0, posinf=8.0),
                       torch.where(sees(n - 3), 7.0, torch.where(sees(7), 8.0, clean[..., 19])))
    keep = [d for d in range(D) if d not in (16, 17, 18, 19)]
    assert torch.equal(got[..., keep], clean[..., keep])


@pytest.mark.parametrize("lo,hi", [(64, 192), (5, 133), (1, 129)])
def test_a_given_output_may_have_any_strides(lo, hi):
    """Rows that begin anywhere, as in the cache's attend; what lies between
    them and the rows past the last sequence are left alone."""
    from innerq_b200.prompt import prompt_attention
    n = [130, 31]
    q, k, v = data([170], [170], 4, 2, "fp16", seed=25)
    want = prompt_attention(q, k, v, cu(n))[:161]
    wide = torch.full((170, 4, 257), 3.0, dtype=torch.float16, device="cuda")
    out = wide[..., lo:hi]
    assert prompt_attention(q, k, v, cu(n), out=out) is not None
    assert torch.equal(out[:161], want)
    assert (wide[161:] == 3).all() and (wide[..., :lo] == 3).all() and (wide[..., hi:] == 3).all()


def test_an_output_whose_rows_overlap_is_refused():
    from innerq_b200.paged import PagedCache
    from innerq_b200.prompt import prompt_attention
    q, k, v = data([3], [3], 4, 2, "fp16")
    with pytest.raises(ValueError):
        prompt_attention(q, k, v, cu([3]), out=torch.zeros((3, 1, D), dtype=torch.float16, device="cuda").expand(3, 4, D))
    c = PagedCache.allocate(1, 2, 3, 32, 0, 32)
    i32 = torch.zeros(3, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        c.attend(q, i32[:, None], i32, i32, out=torch.zeros((1, 4, D), dtype=torch.float16, device="cuda").expand(3, 4, D))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("nq,nk,hq,hkv", [([900, 40], [900, 40], 4, 2), ([1030], [1030], 5, 1), ([2500, 1, 1301], [2500, 1, 1301], 2, 1),
                                          ([300, 77], [4000, 1205], 4, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_every_key_counts_once(nq, nk, hq, hkv, causal, dtype):
    """Bounds that shrink with the context: an element's error is at most the
    output's rounding and that of the probabilities, in sum p |v|.  Where at
    least 100 keys share the weight the latter is a random walk, of steps of at
    most the type's half step / sqrt 3 of p v, and a row's root mean square
    stays within 1.35 of both together (128 channels scatter by a sixteenth; the
    largest of some ten thousand rows by five of those): a single key missed or taken twice is several times
    that.  The log-sum-exp is within 1e-4."""
    from innerq_b200.prompt import prompt_attention
    q, k, v = data(nq, nk, hq, hkv, dtype, seed=27)
    q *= 0.5
    lse = torch.empty(q.shape[:2], device="cuda")
    out = prompt_attention(q, k, v, cu(nq), cu(nk), causal=causal, lse=lse).double()
    R, o, x = hq // hkv, 0, 0
    for a, b in zip(nq, nk):
        i, j = torch.arange(a, device="cuda")[:, None], torch.arange(b, device="cuda")
        for h in range(hq):
            vv = v[x:x + b, h // R].double()
            s = q[o:o + a, h].double() @ k[x:x + b, h // R].double().T * D ** -0.5
            if causal:
                s = s.masked_fill(j > i + b - a, float("-inf"))
            p = torch.softmax(s, -1)
            want = p @ vv
            err = (out[o:o + a, h] - want).abs()
            assert float((lse[o:o + a, h].double() - torch.logsumexp(s, -1) / np.log(2.0)).abs().max()) < 1e-4
            assert bool((err <= ULP[dtype] * (want.abs() * 1.01 + p @ vv.abs()) + 1e-6).all())
            walk = (p.square() @ vv.square()).sqrt()
            expect = ((ULP[dtype] * want).square() + (ULP[dtype] * walk).square()).mean(-1).div(3).sqrt()
            many = p.square().sum(-1) < 0.01
            assert bool((err.square().mean(-1).sqrt() <= 1.35 * expect + 1e-6)[many].all())
        o, x = o + a, x + b


@pytest.mark.parametrize("n,nk", [(40, 30), (300, 290)])
def test_a_scale_that_is_not_a_number(n, nk):
    """NaN for every query that sees a key, as in the cache's attend, zeros for
    the others."""
    from innerq_b200.prompt import prompt_attention
    q, k, v = data([n], [nk], 4, 2, "fp16", seed=28)
    lse = torch.zeros(q.shape[:2], device="cuda")
    out = prompt_attention(q, k, v, cu([n]), cu([nk]), scale=float("nan"), lse=lse)
    assert torch.isnan(out[10:]).all() and torch.isnan(lse[10:]).all()
    assert (out[:10] == 0).all() and torch.isneginf(lse[:10]).all()
