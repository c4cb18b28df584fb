"""What ScoredRouter, BlockNorm, Sampler and their callers hand to the library: host code only, no GPU.  OnGpu stands
for a tensor of a GPU: its address is never read."""
import pytest
import torch

from moe_prefetch import MoeCache, block, lib
from moe_prefetch.batched import BatchedMoe
from moe_prefetch.block import BlockNorm, Sampler, ScoredRouter

F32 = torch.float32


class Memory:
    """What a tensor's address points to."""


class OnGpu:
    """A tensor's shape, strides and dtype, said to be on cuda:<device> at `at`, in memory that its aliases share."""

    is_cuda = True

    def __init__(self, *shape, dtype=F32, device=0, at=4096):
        self._t, self._at, self.device = torch.empty(shape, dtype=dtype, device="meta"), at, torch.device("cuda", device)
        self.memory = Memory()

    def __getattr__(self, name):
        return getattr(self._t, name)

    def __getitem__(self, rows):
        t = OnGpu(dtype=self.dtype, device=self.device.index, at=self._at)
        t._t, t.memory = self._t[rows], self.memory
        return t

    def detach(self):
        return self[...]

    def get_device(self):
        return self.device.index

    def data_ptr(self):
        return self._at


@pytest.fixture
def cache():
    c = MoeCache(2, n_experts=128, intermediate=768, n_slots=16, device=-1)
    yield c
    c.close()


# ---- a cache's scoring rule ---------------------------------------------------------
def test_a_cpu_bias_is_refused():
    with pytest.raises(ValueError, match="bias is on cpu, not on a GPU"):
        ScoredRouter(128, 8, bias=torch.zeros(128))


@pytest.mark.parametrize("bias", [torch.zeros(128), OnGpu(127), OnGpu(128, dtype=torch.bfloat16), OnGpu(256)[::2]])
def test_a_rule_checks_the_bias_that_it_hands_on(cache, bias):
    # the bias may be exchanged for another tensor after the router was made
    router = ScoredRouter(128, 8, bias=OnGpu(128))
    router.bias = bias
    with pytest.raises(ValueError, match="bias"):
        router.rule()
    with pytest.raises(ValueError, match="bias"):
        cache.set_scoring(0, router)


def test_a_cache_takes_a_bias_of_its_own_gpu_alone(cache):
    cache.device = 1                                  # (the library's part of it has none)
    with pytest.raises(ValueError, match="bias is on cuda:0"):
        cache.set_scoring(0, ScoredRouter(128, 8, bias=OnGpu(128)))
    cache.set_scoring(0, ScoredRouter(128, 8, bias=OnGpu(128, device=1)))


def test_a_cache_keeps_the_bias_that_it_reads(cache):
    import gc
    import weakref
    router = ScoredRouter(128, 8, bias=OnGpu(128))
    given = weakref.ref(router.bias.memory)
    cache.set_scoring(0, router)
    router.bias.memory = Memory()                     # as an assignment to a tensor's data
    router.bias = OnGpu(128, at=8192)                 # of the router's own calls from here on
    gc.collect()
    assert given() is not None
    cache.set_scoring(0, router)
    gc.collect()
    assert given() is None
    given = weakref.ref(router.bias.memory)
    cache.set_scoring(0, None)
    del router
    gc.collect()
    assert given() is None


# ---- what a call hands to the library -------------------------------------------------
class Calls:
    """In place of an entry point: notes the descriptor and the stream of each call."""

    def __init__(self):
        self.seen = []

    def __call__(self, desc, stream):
        self.seen.append((desc, stream))
        return 0


@pytest.fixture
def on_device_0(monkeypatch):
    monkeypatch.setattr(block, "_device", lambda: 0)
    monkeypatch.setattr(block, "_raw_stream", lambda dev: 77)


def noted(obj):
    obj._fn = Calls()
    return obj, obj._fn.seen


def product(T=5, E=128, K=8, ws=None, **kw):
    """A call of from_product, as BatchedMoe.route makes it."""
    router, seen = noted(ScoredRouter(E, K))
    ws = OnGpu(lib().moe_route_workspace_bytes(E, T), dtype=torch.uint8) if ws is None else ws
    a = dict(W=OnGpu(E, 2048), x=OnGpu(T, 2048), ids=OnGpu(T, K, dtype=torch.int32), w=OnGpu(T, K),
             slots=OnGpu(T, K, dtype=torch.int32), workspace=ws, H=2048)
    router.from_product(**{**a, **kw})
    return seen


def test_the_routers_product_checks_its_workspace(on_device_0):
    size = lib().moe_route_workspace_bytes(128, 5)
    assert size > 5 * 128 * 4
    for ws in (None, OnGpu(size + 256, dtype=torch.uint8), OnGpu(size // 4), OnGpu(2, size // 8)):
        assert len(product(ws=ws)) == 1
    for ws in (OnGpu(size - 1, dtype=torch.uint8), OnGpu(size // 4 - 1), OnGpu(0), OnGpu(2 * size, dtype=torch.uint8)[::2],
               OnGpu(size, dtype=torch.uint8, device=1), torch.zeros(size, dtype=torch.uint8)):
        with pytest.raises(ValueError, match="workspace"):
            product(ws=ws)


def layer(T=5, E=128, K=8):
    """A BatchedMoe without its device memory."""
    m = BatchedMoe.__new__(BatchedMoe)
    m.T, m.E, m.K, m.H = T, E, K, 2048
    m.ids, m.w, m.slots = OnGpu(T, K, dtype=torch.int32), OnGpu(T, K), OnGpu(T, K, dtype=torch.int32)
    m.route_ws = OnGpu(lib().moe_route_workspace_bytes(E, T), dtype=torch.uint8)
    return m


def test_a_scored_layer_names_the_operand_that_is_missing(on_device_0):
    m, (router, seen) = layer(), noted(ScoredRouter(128, 8))
    W, x, logits = OnGpu(128, 2048), OnGpu(5, 2048), OnGpu(5, 128)
    m.route(5, W=W, x=x, router=router)
    m.route(3, logits=logits[:3], router=router)
    assert len(seen) == 2
    for given in (dict(), dict(W=W), dict(x=x), dict(logits=4096), dict(W=4096, x=x), dict(W=W, x=4096)):
        with pytest.raises(ValueError, match="takes logits, or W and x, as tensors"):
            m.route(5, router=router, **given)
    with pytest.raises(ValueError, match="takes logits, or W and x, as tensors"):
        m.forward(OnGpu(5, 2048, dtype=torch.bfloat16), None, 0, 0, 0, 12, W=W, router=router)
    for given in (dict(logits=logits[:3]), dict(W=W, x=x[:3]), dict(W=W[:64], x=x)):
        with pytest.raises(ValueError):
            m.route(5, router=router, **given)
    assert len(seen) == 2


class Stream:
    def __init__(self, device, handle=55):
        self.device, self.cuda_stream = torch.device("cuda", device), handle


def test_a_stream_of_another_device_is_refused(on_device_0, monkeypatch):
    # (the kernels would run there, on memory and with outputs of this one)
    monkeypatch.setattr(block, "_empty", lambda shape, dtype, dev, stream: OnGpu(*shape, dtype=dtype))
    calls = []
    router, norm, sampler = ScoredRouter(64, 8), BlockNorm(64), Sampler(64)
    for obj, args in ((router, (OnGpu(3, 64),)), (norm, (OnGpu(3, 64),)), (sampler, (OnGpu(3, 64), OnGpu(3)))):
        obj, seen = noted(obj)
        with pytest.raises(ValueError, match="stream is of cuda:1, the call's tensors on cuda:0"):
            obj(*args, stream=Stream(1))
        assert not seen
        obj(*args, stream=Stream(0))
        obj(*args, stream=66)
        obj(*args)
        assert [s for _, s in seen] == [55, 66, 77]
        calls += seen
    m, (router, seen) = layer(), noted(ScoredRouter(128, 8))
    with pytest.raises(ValueError, match="stream is of cuda:1"):
        m.route(5, W=OnGpu(128, 2048), x=OnGpu(5, 2048), router=router, stream=Stream(1))
    m.route(5, W=OnGpu(128, 2048), x=OnGpu(5, 2048), router=router)
    assert [s for _, s in seen] == [0]


def test_outputs_are_not_allocated_on_a_refused_stream(on_device_0, monkeypatch):
    monkeypatch.setattr(block.torch.cuda, "stream", lambda s: pytest.fail("entered"))
    with pytest.raises(ValueError, match="stream is of cuda:1"):
        Sampler(64)(OnGpu(3, 64), OnGpu(3), stream=Stream(1))


def test_a_norm_keeps_the_memory_of_its_weights():
    import gc
    import weakref
    given = [OnGpu(64) for _ in range(4)]
    norm = BlockNorm(64, *given)
    held = [weakref.ref(t.memory) for t in given]
    for t in given:
        t.memory = Memory()                           # as an assignment to a parameter's data: the address stays the norm's
    del given, t
    gc.collect()
    assert all(h() is not None for h in held)
    del norm
    gc.collect()
    assert all(h() is None for h in held)
