"""GPU tests of page copies: every byte of the cache is compared."""
import pytest
import torch

from augur_v100_b200 import host, kv

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def stream():
    torch.cuda.set_device(0)
    s = host.Stream(0)
    yield s
    s.close()


def _cache(layers, pages, kv_heads, page_tokens, head_dim, seed=0):
    g = torch.Generator(device="cuda:0").manual_seed(seed)
    shape = (layers, pages, kv_heads, page_tokens, head_dim)
    bits = lambda: torch.randint(-2 ** 15, 2 ** 15, shape, generator=g, device="cuda:0", dtype=torch.int16)  # noqa: E731
    return kv.KvCache(bits().view(torch.bfloat16), bits().view(torch.bfloat16))


def _same(cache, keys, values):
    return torch.equal(cache.keys.view(torch.int16), keys) and torch.equal(cache.values.view(torch.int16), values)


@pytest.mark.parametrize("layers,kv_heads,page_tokens,head_dim", [(1, 1, 16, 128), (3, 4, 64, 256), (2, 3, 16, 128), (1, 7, 1024, 128), (5, 1, 32, 128)])
@pytest.mark.parametrize("pairs", [1, 2, 7])
def test_copies(stream, layers, kv_heads, page_tokens, head_dim, pairs):
    cache = _cache(layers, 17, kv_heads, page_tokens, head_dim, pairs)
    keys, values = cache.keys.view(torch.int16).clone(), cache.values.view(torch.int16).clone()
    order = torch.randperm(17, generator=torch.Generator().manual_seed(pairs)).tolist()
    sources, destinations = order[:pairs], order[pairs:2 * pairs]
    kv.KvPageCopy.bind(stream, cache).submit(sources, destinations)
    stream.synchronize()
    keys[:, destinations], values[:, destinations] = keys[:, sources], values[:, sources]
    assert _same(cache, keys, values)


def test_lists_longer_than_a_launch_and_one_source_for_many(stream):
    cache = _cache(2, 5003, 1, 16, 128)
    keys, values = cache.keys.view(torch.int16).clone(), cache.values.view(torch.int16).clone()
    order = torch.randperm(5003, generator=torch.Generator().manual_seed(1)).tolist()
    sources, destinations = order[:2300] + [order[0]] * 150, order[2300:4750]
    copy = kv.KvPageCopy.bind(stream, cache)
    copy.submit(sources, destinations)
    stream.synchronize()
    keys[:, destinations], values[:, destinations] = keys[:, sources], values[:, sources]
    assert _same(cache, keys, values)
    launches = host.launch_count()
    copy.submit([], [])
    for bad in (([1], [1]), ([1, 2], [3, 3]), ([1, 2], [2, 3])):
        with pytest.raises(host.CudaRuntimeError):
            copy.submit(*bad)
    for bad in (([1], []), ([-1], [2]), ([1], [5003])):
        with pytest.raises(ValueError):
            copy.submit(*bad)
    stream.synchronize()
    assert host.launch_count() == launches and _same(cache, keys, values)


def test_copies_stay_in_order_with_a_replay_behind_them(stream):
    # a chain a -> b, b -> c over two submits, captured: the second sees what the first wrote
    side = host.Stream(0, torch.cuda.Stream())
    cache = _cache(4, 9, 4, 64, 256, 3)
    copy = kv.KvPageCopy.bind(side, cache)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side.torch_stream):
        copy.submit([0, 1], [2, 3])
        copy.submit([2, 3], [4, 5])
    for seed in range(3):
        cache.keys.copy_(_cache(4, 9, 4, 64, 256, seed + 10).keys)
        keys, values = cache.keys.view(torch.int16).clone(), cache.values.view(torch.int16).clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for t in (keys, values):
            t[:, [2, 3]] = t[:, [0, 1]]
            t[:, [4, 5]] = t[:, [0, 1]]
        assert _same(cache, keys, values)
    del graph
    side.close()


def test_refused_caches(stream):
    good = _cache(1, 4, 2, 16, 128)
    for keys, values in ((good.keys, good.values[:, :3]), (good.keys.float(), good.values), (good.keys[..., ::2], good.values[..., ::2]), (good.keys[0], good.values[0]),
                         (good.keys, good.values.cpu())):
        with pytest.raises(ValueError):
            kv.KvCache(keys, values)
    with pytest.raises(host.CudaRuntimeError):
        kv.KvPageCopy.bind(stream, kv.KvCache(good.keys, good.keys))         # one tensor for both
