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


def test_collate_scans_keeps_a_teachers_predicates():
    from scene_graph_prediction.scene_graph_helpers.dataset.synthetic import collate_scans
    scans = [scan(3, 1), scan(2, 2), scan(4, 3)]
    batch = collate_scans(scans)
    for got, parts in zip(batch["teacher_rels"], zip(*[s["teacher_rels"] for s in scans])):
        assert torch.equal(got, torch.cat(parts)) and got.size(0) == batch["rel_points"].size(0)
    plain = [{k: v for k, v in s.items() if k != "teacher_rels"} for s in scans]
    assert "teacher_rels" not in collate_scans(plain)
    assert "teacher_rels" not in collate_scans([dict(s, teacher_rels=None) for s in plain])
    with pytest.raises(ValueError, match="teacher_rels"):
        collate_scans([scans[0], plain[1]])
    with pytest.raises(ValueError, match="teacher_rels"):
        collate_scans([scans[0], scan(3, 4, k=3)])
