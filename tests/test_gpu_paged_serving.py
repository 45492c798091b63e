"""The serving example: chunked prompts and decode steps of a mixed batch give
the logits of the same decoder with plain attention over what the cache holds."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_batched_serving_matches_plain_attention(dtype):
    from examples.paged_serving import Decoder, Server
    model = Decoder(layers=2, heads=6, kv_heads=2, hidden=256, vocab=200, max_pos=1024, dtype=dtype, seed=1)
    server = Server(model, n_pages=40, n_slots=3, page_size=64, w_sink=32, w_recent=32, chunk=100)
    g = torch.Generator().manual_seed(2)
    lens = [1, 260, 33, 100, 217]
    rs = [server.submit(torch.randint(0, 200, (n,), generator=g).tolist(), 12) for n in lens]

    def plain(r):
        """Logits of r's last token, decoded alone: 32-bit attention over the cache's own content."""
        def attend(layer, q, k, v):
            c = server.caches[layer]
            table, slots, n = server._batch([r])
            zero = torch.zeros_like(n)
            cu = torch.tensor([0, r.cached], dtype=torch.int32, device="cuda")
            ck, cv = c.read(table, slots, n, zero, cu, r.cached)
            pos = r.cached - 1
            cos, sin = model.cos[pos], model.sin[pos]
            x = q.float()
            a, b = x[..., :64], x[..., 64:]
            x = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(dtype).float()[0]
            kk, vv = (t.float().repeat_interleave(3, 1).transpose(0, 1) for t in (ck, cv))
            p = torch.softmax((x[:, None] @ kk.transpose(1, 2)) * 128 ** -0.5, -1)
            return (p @ vv).transpose(0, 1).to(dtype)
        return model.forward(torch.tensor([r.tokens[r.cached - 1]], device="cuda"), attend)[0]

    seen = {}
    while server.running or server.waiting:
        before = {id(r): r.cached for r in server.running}
        for r, logits in server.step():
            seen[id(r)] = seen.get(id(r), 0) + 1
            if before.get(id(r), 0) >= r.prompt_len and r.left > 0:
                # a decode step: check against the plain attention (the slot and pages are still r's)
                tok = r.tokens.pop()
                want = plain(r)
                r.tokens.append(tok)
                # 2 layers of type-rounded activations on both sides: a few steps of the type of the largest logit
                tol = (2.0 ** -8 if dtype == torch.float16 else 2.0 ** -5) * float(want.float().abs().max())
                assert float((logits.float() - want.float()).abs().max()) <= tol
    assert all(seen[id(r)] == 12 and len(r.tokens) == n + 12 for r, n in zip(rs, lens))
    assert len(server.free_pages) == 40 and len(server.free_slots) == 3


def test_prompts_in_chunks_match_whole_prompts():
    """A prompt that stays in the 16-bit sink and window gives the same logits in one chunk as in several."""
    from examples.paged_serving import Decoder, Server
    model = Decoder(layers=2, heads=4, kv_heads=1, hidden=256, vocab=100, max_pos=512, dtype=torch.float16, seed=3)
    g = torch.Generator().manual_seed(4)
    prompt = torch.randint(0, 100, (150,), generator=g).tolist()
    out = []
    for chunk in (1024, 64, 37):
        s = Server(model, n_pages=4, n_slots=1, page_size=32, w_sink=32, w_recent=128, chunk=chunk)
        s.submit(prompt, 1)
        got = []
        while s.running or s.waiting:
            got += s.step()
        out.append(got[0][1].float())
    for o in out[1:]:
        # the same products in another order: a few steps of fp16 of the largest logit
        assert float((o - out[0]).abs().max()) <= 2.0 ** -8 * float(out[0].abs().max())


def test_requests_that_can_never_be_served_are_refused():
    """A request without tokens, or that needs more pages or positions than
    there are, would wait for ever and everything behind it too."""
    from examples.paged_serving import Decoder, Server
    model = Decoder(layers=1, heads=2, kv_heads=1, hidden=64, vocab=50, max_pos=300, dtype=torch.float16, seed=5)
    s = Server(model, n_pages=4, n_slots=2, page_size=32, w_sink=32, w_recent=32, chunk=64)
    for prompt, new in (([], 4), ([1], 0), ([1] * 150, 100), ([1] * 290, 12)):
        with pytest.raises(ValueError):
            s.submit(prompt, new)
    assert not s.waiting
    r = s.submit([1] * 150, 45)  # 195 tokens, 128 of them packed: all four pages
    for _ in range(60):
        s.step()
    assert len(r.tokens) == 195 and not s.running and len(s.free_pages) == 4
