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


def plain_distill(logits, index, values, temperature=1.0):
    """distill_top_k's formula in torch."""
    lq = torch.log_softmax(values / temperature, -1)
    lp = torch.log_softmax(logits / temperature, -1).gather(-1, index)
    return temperature ** 2 * (lq.exp() * (lq - lp)).sum(-1)


def per_scan_and_collated(device, dtype):
    """(losses and gradients of scans of 12, 2 and 6 edges one by one: their means, those of the collated batch)"""
    from scene_graph_prediction import main as runner
    from scene_graph_prediction.scene_graph_helpers.dataset.synthetic import collate_scans
    config = runner.config_loader("no_gt.json")
    config["MODEL"]["distill_temperature"], config["MODEL"]["lambda_distill"] = 2.0, 0.5
    model = runner.SGPNModelWrapper(config, 12, 15, torch.ones(12), torch.linspace(0.5, 2, 15), runner.RELATION_NAMES)
    model.weights_obj, model.weights_rel = model.weights_obj.to(dtype), model.weights_rel.to(dtype)
    scans = [scan(4, 1), scan(2, 2), scan(3, 3)]
    gen = torch.Generator().manual_seed(0)
    preds = [[torch.randn(s[k].size(0), n, generator=gen).log_softmax(1).to(device, dtype).requires_grad_()
              for k, n in (("gt_class", 12), ("gt_rels", 15))] for s in scans]
    losses = [model.loss(o, r, to_device(s, device)) for (o, r), s in zip(preds, scans)]
    mean = sum(losses) / 3
    alone = torch.autograd.grad(mean, [p for pair in preds for p in pair])
    batch = to_device(collate_scans(scans), device)
    leaves = [[p.detach().requires_grad_() for p in pair] for pair in preds]
    loss = model.loss(torch.cat([o for o, _ in leaves]), torch.cat([r for _, r in leaves]), batch)
    return (mean, *alone), (loss, *torch.autograd.grad(loss, [p for pair in leaves for p in pair]))


def test_a_batch_of_scans_learns_from_a_teacher_as_its_scans_do(monkeypatch):
    """In 64 bits, with the formula in the kernel's place: equal up to the order of sums of at most 20 terms."""
    from pointnet2_ops import head_ops
    monkeypatch.setattr(head_ops, "distill_top_k", lambda x, i, v, t: plain_distill(x, i, v.to(x.dtype), t))
    for a, b in zip(*per_scan_and_collated("cpu", torch.float64)):
        torch.testing.assert_close(a, b, rtol=1e-12, atol=1e-14)


@pytest.mark.gpu
def test_a_batch_of_scans_learns_from_a_teacher_as_its_scans_do_on_the_gpu():
    """The kernels in fp32: rows are the same in both, the means differ by the order of at most 20 roundings."""
    for a, b in zip(*per_scan_and_collated("cuda", torch.float32)):
        torch.testing.assert_close(a, b, rtol=32 * 2.0 ** -24, atol=32 * 2.0 ** -24 * float(a.detach().abs().max()))


@pytest.mark.gpu
def test_a_teacher_model_and_its_student():
    """teacher_relations of one model is what another one's batch carries: the teacher's best predicates, and a training step with
    them (two scans of different sizes) whose loss is the plain one plus the distillation term of the same forward pass."""
    from scene_graph_prediction import main as runner
    from scene_graph_prediction.scene_graph_helpers.dataset.synthetic import collate_scans
    config = runner.config_loader("no_gt.json")
    torch.manual_seed(3)
    teacher, student = (runner.SGPNModelWrapper(config, 12, 15, torch.ones(12), torch.ones(15), runner.RELATION_NAMES).cuda() for _ in range(2))
    teacher.eval()
    scans = [synthetic_scan(n, 512, 1024, seed=n, scan_id=f"s{n}") for n in (4, 3)]
    for s in scans:
        batch = to_device(s, "cuda")
        s["teacher_rels"] = index, value = teacher.teacher_relations(batch, 4)
        with torch.no_grad():
            best = teacher(batch)[1].topk(4, 1)
        assert index.shape == (s["gt_rels"].numel(), 4) and not value.requires_grad
        assert torch.equal(index, best.indices)
        torch.testing.assert_close(value, best.values, rtol=0, atol=16 * 2.0 ** -24 * (1 + float(best.values.abs().max())))
    student.train()
    batch = to_device(collate_scans(scans), "cuda")
    obj, rel = student(batch)
    loss, plain = student.loss(obj, rel, batch), student.loss(obj, rel, {k: v for k, v in batch.items() if k != "teacher_rels"})
    rows = plain_distill(rel.double(), batch["teacher_rels"][0], batch["teacher_rels"][1].double())
    want = (rows[:12].mean() + rows[12:].mean()) / 2
    assert abs(float((loss - plain - want).detach())) <= 64 * 2.0 ** -24 * float(loss.detach())
    grads = torch.autograd.grad(loss, [p for p in student.rel_predictor.parameters()])
    assert all(g.isfinite().all() and g.any() for g in grads if g.numel())
    student.training_step(batch).backward()


@pytest.mark.gpu
def test_a_replayed_step_reads_its_batch_s_teacher():
    """Whole steps on one batch of scans with learning rate 0 and no dropout: the eager first one, the captured one, replays with other
    predicates of the teacher; every loss is the eager loss of its batch (atomics in the encoders' backward do not reach it)."""
    from runtime import GraphedTrainStep
    from scene_graph_prediction import main as runner
    from scene_graph_prediction.scene_graph_helpers.dataset.synthetic import collate_scans
    torch.manual_seed(4)
    model = runner.SGPNModelWrapper(runner.config_loader("no_gt.json"), 12, 15, torch.ones(12), torch.ones(15), runner.RELATION_NAMES).cuda().train()
    for m in model.modules():
        if isinstance(m, torch.nn.Dropout):
            m.p = 0.0
    for n, p in model.named_parameters():
        if ".backbone.fc_layer." in n:
            p.requires_grad_(False)
    opt = torch.optim.AdamW([p for p in model.parameters() if p.requires_grad], lr=0.0, weight_decay=0.0, capturable=True)
    step = GraphedTrainStep(model.pure_training_step, model.parameters(), opt)

    def batch(seed):
        scans = [dict(synthetic_scan(n, 512, 1024, seed=n, scan_id=f"s{n}"), teacher_rels=scan(n, seed)["teacher_rels"]) for n in (4, 3)]
        return to_device(collate_scans(scans), "cuda")
    losses = []
    for seed in (1, 1, 2, 3, 1):
        b = batch(seed)
        with torch.no_grad():
            want = float(model.pure_training_step(b)[0])
        losses.append(float(step(b)[0]))
        assert abs(losses[-1] - want) <= 1e-5 * want
    assert step.num_graphs == 1 and len({round(v, 4) for v in losses}) == 3
