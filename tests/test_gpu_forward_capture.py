"""Forward calls while the context's stream is being captured: refused before they do anything, and the capture goes on."""
import importlib

import numpy as np
import pytest

from oracle import forward as ofw

pytestmark = pytest.mark.gpu


def test_refused_inside_a_capture(dpb):
    import torch
    fw = importlib.import_module("deep_prove_b200.forward")
    ctx = dpb.Context(0)
    try:
        rng = np.random.default_rng(1)
        E, keys = rng.integers(-99, 99, size=(8, 8)), np.array([1, 0, 1])
        x, W = rng.integers(-99, 99, size=(3, 6)), rng.integers(-99, 99, size=(2, 6, 5))
        table, dev_keys, dev_x = ctx.upload_ints(E.reshape(-1), dpb.FR_I32), ctx.upload_tensor_i64(keys), ctx.upload_tensor_i64(x)
        dev_w = ctx.upload_tensor_i64(W)
        groups, weights = fw.RowGroups(ctx, keys, 2), fw.ExpertWeights(ctx, W, 8)
        eq = ctx.upload(np.ones((4, 2), np.uint64), dpb.GL_EXT)
        many = np.zeros(5000, np.int64)
        calls = [lambda: fw.embedding_lookup(ctx, table, 8, 8, keys), lambda: fw.embedding_lookup(ctx, table, 8, 8, many[:0]),
                 lambda: fw.embedding_lookup(ctx, table, 8, 8, None, device_tokens=dev_keys),
                 lambda: fw.RowGroups(ctx, keys, 2), lambda: fw.RowGroups(ctx, None, 2, device_keys=dev_keys),
                 lambda: fw.RowGroups(ctx, many, 2), lambda: groups.sums(dpb.GL_EXT), lambda: groups.sums(dpb.FR, rows=x),
                 lambda: groups.sums(dpb.GL_EXT, weights=eq, device_rows=dev_x),
                 lambda: fw.ExpertWeights(ctx, W, 8), lambda: fw.ExpertWeights(ctx, None, 8, device_weights=dev_w),
                 lambda: fw.grouped_product(ctx, groups, x, 8, weights),
                 lambda: fw.grouped_product(ctx, groups, None, 8, weights, device_x=dev_x)]
        ctx.sync()
        counter = torch.zeros(4, dtype=torch.int64, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=torch.cuda.ExternalStream(ctx.stream), capture_error_mode="thread_local"):
            counter += 1
            for f in calls:
                with pytest.raises(dpb.DpbError, match="outside captures") as e:
                    f()
                assert e.value.code == dpb.ESTATE
            counter += 1
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        assert counter.tolist() == [6] * 4
        for f in calls:  # and outside they are made
            f()
        y, shape = fw.grouped_product(ctx, groups, x, 8, weights)
        assert np.array_equal(y.to_host(n=15).reshape(shape), ofw.grouped_product(x, keys, W))
        assert groups.sums(dpb.GL_EXT).to_host()[:, 0].tolist() == [1, 2]
        del graph
    finally:
        ctx.close()
