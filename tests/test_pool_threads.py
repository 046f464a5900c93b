"""A pool that several threads use first at the same time makes its tensors once, and no thread sees a part."""

from __future__ import annotations

import threading

import pytest
import torch

from runtime_amd.phase2.paged_kv_kernel import GpuKVBlockPool


class _Interrupted(GpuKVBlockPool):
    """Another thread asks for a layer after every attribute that the first use sets."""

    def __setattr__(self, name, value):
        super().__setattr__(name, value)
        if getattr(self, "asking", None) is not None and threading.current_thread() is threading.main_thread():
            thread = threading.Thread(target=self.ask)
            self.asking.append(thread)
            thread.start()
            thread.join(0.05)  # it either answers or waits for the first

    def ask(self):
        try:
            self.answers.append(self.k_layer_view(1).data_ptr())
        except Exception as e:  # noqa: BLE001 - what a worker thread would die of
            self.answers.append(e)


@pytest.mark.parametrize("layout", ["interleaved", "split"])
def test_first_use_from_several_threads(layout):
    pool = _Interrupted(num_blocks=3, block_size_tokens=4, num_layers=2, num_kv_heads=1, head_dim=8,
                        dtype=torch.float32, device="cpu", kv_layout=layout)
    object.__setattr__(pool, "answers", [])
    object.__setattr__(pool, "asking", [])
    first = pool.k_layer_view(1)
    for thread in pool.asking:
        thread.join(10)
    assert len(pool.answers) == len(pool.asking) >= 4
    assert pool.answers == [first.data_ptr()] * len(pool.answers), pool.answers
