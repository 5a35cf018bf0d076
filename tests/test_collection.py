"""What tests/conftest.py decides about the collected tests."""
import os

import pytest
import torch

from tests import conftest


class Item:
    def __init__(self, module, name='test'):
        self.fspath, self.name, self.marks = os.path.join('tests', module + '.py'), name, []

    def add_marker(self, mark):
        self.marks.append(mark.name)


def collect(*items):
    items = list(items)
    conftest.pytest_collection_modifyitems(None, None, items)
    return items


@pytest.mark.parametrize('gpu', [False, True])
def test_host_only_tests_do_not_meet_a_gpu(monkeypatch, gpu):
    monkeypatch.setattr(torch.cuda, 'is_available', lambda: gpu)
    items = collect(Item('test_learn_ops_host'), Item('test_learn_ops_limits'), Item('test_mesh'))
    assert {(i.fspath.split(os.sep)[-1], tuple(i.marks)) for i in items} == {
        ('test_learn_ops_host.py', ('skip',) if gpu else ()), ('test_learn_ops_limits.py', ('skip',) if gpu else ()), ('test_mesh.py', ())}


def test_what_needs_files_from_outside_runs_last():
    names = [i.name for i in collect(Item('test_gpu_chain', 'test_oracle_is_pinned_on_this_box'), Item('test_gpu_fullsize', 'a'), Item('test_gpu_learn_scan', 'b'),
                                     Item('test_gpu_ops', 'c'))]
    assert names == ['c', 'b', 'a', 'test_oracle_is_pinned_on_this_box']
