"""Recorded attention calls and the device whose workspace they use."""
import numpy as np
import pytest

import attention_ref as ref

pytestmark = pytest.mark.gpu


def recorded(dev, rng):
    """an attention whose keys are shared out over blocks, recorded; its buffers, which stay in use"""
    p = ref.Paged(rng, "f16", 4, 2, 64, 16, [900], [1])
    cache = dev.paged_cache(ref.upload(dev, p.k, "f16"), ref.upload(dev, p.v, "f16"), dev.upload(p.table), dev.upload(p.lens.astype(np.int32)))
    q, starts, out = ref.upload(dev, p.q, "f16"), dev.upload(p.starts), ref.upload(dev, np.zeros(p.q.shape), "f16")
    dev.paged_attention(q, cache, starts, out=out)
    want = out.to_numpy()
    with dev.capture() as graph:
        dev.paged_attention(q, cache, starts, out=out)
    return graph, want, out, (cache, q, starts)


def test_a_graph_does_not_outlive_its_device():
    """devices made later may lie where the first one lay; none of them is taken for it"""
    from ratchet_amd import Device

    rng = np.random.default_rng(0)
    first = Device(0)
    graph, want, out, held = recorded(first, rng)
    out.zero_()
    graph.launch()
    assert np.array_equal(out.to_numpy(), want)
    handle = graph.graph.handle
    first.close()
    for _ in range(20):
        later = Device(0)
        assert later.lib.rt_graph_launch(later.handle, handle) == 7                # RT_ERR_ARG
        later.close()
    assert later.lib.rt_graph_destroy(handle) == 0
    graph.graph.handle = None
