"""What outlives what: graphs over a cache that another has taken the place of, passes on other streams, tensors of a cache that are exchanged."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_paged_decoder_gpu import DEV, _cache, _decoder, _i32, _prompt  # noqa: E402

BITWISE = dict(ffn_profile=(4, 24, 6))   # no kernel whose sums differ in the last bit from call to call


def test_a_graph_over_an_earlier_cache_replays_after_a_larger_one_was_attached():
    """The larger cache outgrows every buffer of the decoder; the older graph still runs on those it was captured with."""
    dec = _decoder(64 * 4, **BITWISE)
    prompt = _i32(np.random.default_rng(1).integers(0, 1000, (1, 7)))
    want = []
    for graphed in (False, True):
        cache = _cache(1, pages=4, width=3)
        dec.set_cache(cache)
        _prompt(dec, cache, prompt)
        token = _i32([3])
        if not graphed:
            for _ in range(20):
                assert int(cache.extend(1)) == 0
                token = dec.step(token)
                want.append((int(token), dec.read_logits(1)))
            continue
        keep = [x.clone() for x in (cache.k, cache.v, cache.table, cache.lens, cache.refs)]
        cache.extend(1)
        dec.step(token)   # once before the capture
        graph, out = torch.cuda.CUDAGraph(), torch.empty_like(token)
        with torch.cuda.graph(graph):
            cache.extend(1)
            dec.step(token, out)
            token.copy_(out)
        for x, y in zip((cache.k, cache.v, cache.table, cache.lens, cache.refs), keep):
            x.copy_(y)
        token.fill_(3)
        large = _cache(4, pages=60, width=10)
        for i in range(20):
            dec.set_cache(large)
            if i == 0:
                _prompt(dec, large, _i32(np.random.default_rng(2).integers(0, 1000, (4, 60))))
            assert int(large.extend(1)) == 0
            dec.step(_i32([5, 6, 7, 8]))
            graph.replay()
            assert int(token) == want[i][0] and torch.equal(dec.read_logits(1), want[i][1]), i
        assert large.lens.tolist() == [80] * 4 and cache.lens.tolist() == [27]
    dec.free()


def test_passes_on_a_side_stream():
    """A cache attached and run on a stream that does not wait for the default one, against the default stream; and a captured verification."""
    dec = _decoder(3 * 64, **BITWISE)
    rng = np.random.default_rng(3)
    prompt, ids = _i32(rng.integers(0, 1000, (3, 20))), _i32(rng.integers(0, 1000, (3, 6)))
    tree = _i32([[-1, 0, 0, 1, 2, 4]] * 3)
    runs = []
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (torch.cuda.current_stream(), side):
        with torch.cuda.stream(stream):
            cache = _cache(3)
            dec.set_cache(cache)
            _prompt(dec, cache, prompt)
            token, out = _i32([1, 2, 3]), []
            for _ in range(10):
                cache.extend(1)
                token = dec.step(token)
                out.append(token)
            cache.extend(6)
            targets = dec.verify(ids, tree)
            kept = cache.accept(ids, tree, targets, lens_out=cache.lens)
            runs.append([torch.stack(out), targets, *kept, cache.k, cache.v, cache.table, dec.read_logits(18)])
        torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    dec.free()


def test_a_cache_attached_and_run_at_once_on_a_side_stream():
    """Nothing between the attachment, whose constants are copied from the host, and the first pass on a stream that waits for no other."""
    tokens, runs = _i32([1, 2, 3]), []
    side = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), side):
        dec = _decoder(8, **BITWISE)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            cache = _cache(3)
            cache.extend(5)
            dec.set_cache(cache)
            steps = [dec.step(tokens) for _ in range(5)]
            runs.append((torch.stack(steps), dec.read_logits(3), cache.k, cache.v))
        torch.cuda.synchronize()
        dec.free()
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_a_captured_verification_replays():
    dec = _decoder(2 * 64, **BITWISE)
    rng = np.random.default_rng(4)
    prompt = _i32(rng.integers(0, 1000, (2, 18)))
    tree = _i32([[-1, 0, 0, 1, 1, 2, 5], [-1, 0, 1, 2, 0, 4, 4]])
    caches = [_cache(2), _cache(2)]
    for c in caches:
        dec.set_cache(c)
        _prompt(dec, c, prompt)
    ids = torch.zeros(2, 7, dtype=torch.int32, device=DEV)

    def step(c):
        lack = c.extend(7)
        targets = dec.verify(ids, tree)
        return (lack, targets, *c.accept(ids, tree, targets, lens_out=c.lens))

    keep = [x.clone() for x in (caches[1].k, caches[1].v, caches[1].table, caches[1].lens, caches[1].refs)]
    step(caches[1])
    for x, y in zip((caches[1].k, caches[1].v, caches[1].table, caches[1].lens, caches[1].refs), keep):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(caches[1])
    for i in range(15):
        ids.copy_(_i32(rng.integers(0, 1000, (2, 7))))
        dec.set_cache(caches[0])
        # half of the drafts are the model's own: what a dry pass says of the root goes to one of its children
        assert int(caches[0].extend(7)) == 0
        if i % 2:
            first = dec.verify(ids, tree)
            ids[:, 1] = first[:, 0]
        want = [x.clone() for x in step(caches[0])]
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(want, outs)), i
        assert int(want[0]) == 0 and torch.equal(caches[0].lens, caches[1].lens)
        if i % 2:
            assert (want[2] >= 2).all()
    assert torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].table, caches[1].table)
    dec.free()


def test_tensors_of_a_cache_are_not_exchanged():
    """The library holds their addresses: another tensor under the same name would not be what the calls work on."""
    cache = _cache(2)
    for name in ("k", "v", "table", "lens", "refs"):
        with pytest.raises(AttributeError, match=name):
            setattr(cache, name, getattr(cache, name).clone())
    lens = cache.lens
    cache.lens += 3   # in place: the same tensor
    assert cache.lens is lens and cache.lens.tolist() == [3, 3]


def test_tokens_with_a_stride():
    """A column of a matrix is a batch of tokens like any other; outputs that a step cannot fill are refused."""
    dec = _decoder(8, max_ctx=40, **BITWISE)
    ids = _i32(np.random.default_rng(5).integers(0, 1000, (3, 8)))
    for paged in (False, True):
        got = []
        for contiguous in (True, False):
            if paged:
                cache = _cache(3)
                dec.set_cache(cache)
                assert int(cache.extend(8)) == 0
            else:
                dec.fill_cache(0)
            run = []
            for i in range(8):
                dec.step(ids[:, i].contiguous() if contiguous else ids[:, i])
                run.append(dec.read_logits(3))
            got.append(torch.stack(run))
        assert torch.equal(*got)
    out = torch.empty(3, 2, dtype=torch.int32, device=DEV)
    for bad in (out[:, 0], out[:2, 0].contiguous(), torch.empty(3, dtype=torch.int64, device=DEV), torch.empty(3, dtype=torch.int32)):
        with pytest.raises(ValueError, match="ids_out"):
            dec.step(ids[:, 0], bad)
    dec.free()
