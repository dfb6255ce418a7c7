"""A batch that carries another model's best predicates (``teacher_rels``) on its way to the loss."""
import pytest
import torch

from scene_graph_prediction.scene_graph_helpers.dataset.synthetic import synthetic_scan, to_device


def scan(n_obj, seed, k=5):
    s = synthetic_scan(n_obj, 16, 24, seed=seed, scan_id=f"s{seed}")
    gen = torch.Generator().manual_seed(seed)
    best = torch.randn(s["rel_points"].size(0), 15, generator=gen).log_softmax(1).topk(k, 1)
    return dict(s, teacher_rels=(best.indices, best.values))


def test_to_device_moves_a_teachers_tensors():
    s = scan(3, 1)
    moved = to_device(s, "meta")
    assert isinstance(moved["teacher_rels"], tuple) and [t.device.type for t in moved["teacher_rels"]] == ["meta"] * 2
    assert moved["obj_points"].device.type == "meta" and moved["objs_json"] is s["objs_json"] and moved["scan_id"] == "s1"
    assert [t.device.type for t in to_device(dict(s, teacher_rels=list(s["teacher_rels"])), "meta")["teacher_rels"]] == ["meta"] * 2
    assert to_device(dict(s, crop=(1, 2)), "meta")["crop"] == (1, 2)
