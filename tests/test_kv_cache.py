"""The streaming layer's cache (``solb200.KVCache``), whose bookkeeping runs on any device."""

import pytest
import torch

import solb200


def _tokens(B, T, start):
    return torch.full((B, T, 1, 2), float(start), dtype=torch.bfloat16) + torch.arange(T)[:, None, None]


def _append(cache, B, T, start):
    k = _tokens(B, T, start)
    cache.append(k, -k)


def test_tokens_go_behind_each_length():
    cache = solb200.KVCache(2, 8, 1, 2, "cpu")
    _append(cache, 2, 3, 0)
    cache.lengths[1] = 1                       # a ragged prompt: the second sequence has one token
    _append(cache, 2, 2, 10)
    assert cache.lengths.tolist() == [5, 3]
    assert cache.k[0, :5, 0, 0].tolist() == [0, 1, 2, 10, 11]
    assert cache.k[1, :3, 0, 0].tolist() == [0, 10, 11]
    assert torch.equal(cache.v[1, :3], -cache.k[1, :3])


@pytest.mark.parametrize("inference", [False, True])
@pytest.mark.parametrize("how", ["appended", "in place", "set"])
def test_past_the_capacity_is_refused_and_changes_nothing(how, inference):
    with torch.inference_mode(inference):
        cache = solb200.KVCache(2, 8, 1, 2, "cpu")
        cache.k.zero_()
        _append(cache, 2, 4, 1)
        if how == "appended":
            _append(cache, 2, 3, 5)
        elif how == "in place":
            cache.lengths[0] = 7
        else:
            cache.lengths = torch.tensor([7, 2], dtype=torch.int32)
        before, k = cache.lengths.clone(), cache.k.clone()
        for _ in range(2):
            with pytest.raises(RuntimeError, match="solb200.*do not fit"):
                _append(cache, 2, 2, 20)
            assert torch.equal(cache.lengths, before) and torch.equal(cache.k, k)
        _append(cache, 2, 1, 30)
        assert cache.k[0, 7, 0, 0] == 30 and cache.lengths[0] == 8
        with pytest.raises(RuntimeError, match="solb200.*do not fit"):
            _append(cache, 2, 1, 40)
        cache.lengths.zero_()                  # started again: room for all of it
        _append(cache, 2, 8, 50)
        assert cache.lengths.tolist() == [8, 8] and cache.k[1, :, 0, 0].tolist() == list(range(50, 58))
        with pytest.raises(RuntimeError, match="solb200.*do not fit"):
            _append(cache, 2, 9, 0)


def test_lengths_are_read_back_only_where_they_have_to_be(monkeypatch):
    cache = solb200.KVCache(1, 6, 1, 2, "cpu")
    reads = []
    most = torch.Tensor.max
    monkeypatch.setattr(torch.Tensor, "max", lambda t, *a: (reads.append(1), most(t, *a))[1])
    for i in range(6):
        _append(cache, 1, 1, i)
    assert not reads
    cache.lengths.fill_(2)
    _append(cache, 1, 1, 7)
    assert len(reads) == 1
    _append(cache, 1, 1, 8)
    assert len(reads) == 1


def test_no_sequences_and_no_tokens():
    _append(solb200.KVCache(0, 4, 1, 2, "cpu"), 0, 3, 0)
    cache = solb200.KVCache(2, 0, 1, 2, "cpu")
    with pytest.raises(RuntimeError, match="solb200.*do not fit"):
        _append(cache, 2, 1, 0)
    cache = solb200.KVCache(2, 2, 1, 2, "cpu")
    _append(cache, 2, 2, 0)
    _append(cache, 2, 0, 0)
    assert cache.lengths.tolist() == [2, 2]


def test_the_cache_keeps_values_not_their_history():
    cache = solb200.KVCache(1, 4, 1, 2, "cpu")
    k = _tokens(1, 2, 0).requires_grad_()
    cache.append(k * 2, k * 3)
    assert not cache.k.requires_grad and not cache.v.requires_grad
    assert cache.k[0, :2, 0, 0].tolist() == [0, 2] and cache.v[0, :2, 0, 0].tolist() == [0, 3]


def test_a_cached_call_refuses_an_input_that_requires_a_gradient():
    layer = solb200.StreamingSelfAttention(16, 1, head_dim=64)
    cache = layer.new_cache(1, 4)
    with pytest.raises(RuntimeError, match="solb200.*gradient"):
        layer(torch.zeros(1, 1, 16, requires_grad=True), torch.zeros(1, 32), torch.zeros(1, 32), cache=cache)
    assert cache.lengths.tolist() == [0]


@pytest.mark.gpu
def test_a_captured_step_past_the_capacity_stays_in_the_cache(cuda_device):
    """Replays read nothing back: past the capacity the last place takes the token, nothing outside
    it is written, and the next plain call refuses."""
    guard = torch.full((3, 6, 1, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    cache = solb200.KVCache(2, 6, 1, 64, "cuda")
    cache.k, cache.v = guard[:2], guard[:2].clone()          # (the third sequence lies right behind)
    token = torch.zeros(2, 1, 1, 64, dtype=torch.bfloat16, device="cuda")
    cache.append(token + 1, token + 1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(token, token)
    for i in range(2, 10):
        token.fill_(i)
        graph.replay()
    torch.cuda.synchronize()
    assert cache.k[1, :, 0, 0].tolist() == [1, 2, 3, 4, 5, 9] and (guard[2] == 7).all()
    assert cache.lengths.tolist() == [9, 9]
    with pytest.raises(RuntimeError, match="solb200.*do not fit"):
        cache.append(token, token)
    cache.lengths.fill_(3)
    cache.append(token, token)
    assert cache.lengths.tolist() == [4, 4] and cache.k[0, 3, 0, 0] == 9


@pytest.mark.gpu
def test_cached_calls_with_gradients_enabled_keep_no_graph(cuda_device):
    """The layer's parameters require gradients: a stream without no_grad() gives the same values and
    leaves neither the cache nor the output with a history."""
    torch.manual_seed(2)
    layer = solb200.StreamingSelfAttention(128, 2, head_dim=64, left=6, sinks=2).cuda()
    layer.qkv.bfloat16()
    layer.out.bfloat16()
    x = torch.randn(2, 5, 128, device="cuda").bfloat16()
    angle = torch.randn(5, 32, device="cuda")
    runs = []
    for enabled in (True, False):
        with torch.set_grad_enabled(enabled):
            cache = layer.new_cache(2, 8)
            cache.k.zero_()
            runs.append([layer(x[:, t:t + 1], angle[t:t + 1].cos(), angle[t:t + 1].sin(), cache=cache) for t in range(5)])
            assert not cache.k.requires_grad and not cache.v.requires_grad
    for a, b in zip(*runs):
        assert torch.equal(a, b) and not a.requires_grad
