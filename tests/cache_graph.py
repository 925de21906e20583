"""A call of the operators around the paged cache recorded into a graph, with the workspace it takes there."""
import contextlib

import torch


@contextlib.contextmanager
def recorded(ops, pkg, call):
    """(graph, what the call returned while it was recorded)"""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(6):                                           # until the allocator has all that a pass asks for
            before = pkg.runtime.cachingStats()["num_device_malloc"]
            warm = ops.WorkspaceScope()
            with warm:
                call()
            side.synchronize()
            warm.close()
            if pkg.runtime.cachingStats()["num_device_malloc"] == before:
                break
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        scope = ops.WorkspaceScope()
        with scope:
            out = call()
    yield graph, out
    del graph
    scope.close()
