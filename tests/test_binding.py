"""The maintainer-side binding snippet of the integration guide is executed as written, on a stand-in for
the reference's model object, and (on a GPU) driven in the order of src/train.py:148-156 / src/test.py:95-99."""
import inspect
import os
import re

import pytest
import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class StandInModel:
    """What bind_boxops needs of the reference's model object: `.nc` (ssd300.py:57: num_classes + 1) and a
    forward that stays the reference's."""

    def __init__(self, nc):
        self.nc = nc

    def forward(self, x):
        return 'network output'

    def loss(self, outputs, gt_bboxes, gt_labels, iou_thresh=0.5, alpha=1.0):
        raise AssertionError('the reference loss must have been replaced')

    def pre_predict(self, outputs, conf_thresh=0.01, top_k=200):
        raise AssertionError('the reference pre_predict must have been replaced')


def integration_snippets():
    text = open(os.path.join(REPO, 'INTEGRATION.md')).read()
    return re.findall(r'```python\n(.*?)```', text, flags=re.S)


def run_binding_snippet(model):
    snip = [s for s in integration_snippets() if 'bind_boxops(model,' in s and 'maintainer-side patch' in s]
    assert len(snip) == 1
    env = {'model': model}
    exec(snip[0], env)                      # noqa: S102 -- the documented snippet, verbatim
    return env['model']


def test_integration_snippet_binds_the_reference_seams():
    import object_detection_amd as D
    m = run_binding_snippet(StandInModel(21))
    assert isinstance(m.boxops, D.SSD300) and m.boxops.nc == 21 and m.boxops.dboxes.shape == (8732, 4)
    assert m.forward(None) == 'network output'                               # the network part is untouched
    # same call signatures as the reference's methods (src/models/ssd300.py:210,339)
    assert list(inspect.signature(m.loss).parameters) == ['outputs', 'gt_bboxes', 'gt_labels', 'iou_thresh', 'alpha']
    assert list(inspect.signature(m.pre_predict).parameters) == ['outputs', 'conf_thresh', 'top_k']
    assert inspect.signature(m.pre_predict).parameters['top_k'].default == 200
    y = D.bind_boxops(StandInModel(20), 'yolov3')                            # yolov3.py: nc = num_classes
    assert y.boxops.nc == 20
    r = D.bind_boxops(StandInModel(81), 'retinanet', f_k_list=[100, 50, 25, 13, 7])
    assert r.boxops.pboxes.shape == (120087, 4)
    assert list(inspect.signature(D.Predictor.run).parameters) == ['self', 'image_metas', 'pred_bboxes', 'pred_scores', 'pred_class_ids']
    assert list(inspect.signature(D.Predictor.__init__).parameters) == ['self', 'iou_thresh', 'classes', 'out_dir']


def test_binding_leaves_a_models_own_head_logits_alone():
    """No GPU needed: a submodule or a method of that name belongs to the network part; without one the box-ops' is bound, and a
    second binding replaces the first's."""
    import object_detection_amd as D

    class WithModule(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.nc = 21
            self.head_logits = torch.nn.Linear(4, 21)

    class WithMethod(StandInModel):
        def head_logits(self, x):
            return 'the network\'s'
    m = WithModule()
    layer = m.head_logits
    assert D.bind_boxops(m, 'ssd300').head_logits is layer and len(list(m.parameters())) == 2
    assert m.boxops.head_logits.__self__ is m.boxops
    assert D.bind_boxops(WithMethod(21), 'ssd300').head_logits(None) == "the network's"
    plain = StandInModel(21)
    for _ in range(2):
        D.bind_boxops(plain, 'ssd300')
        assert plain.head_logits.__self__ is plain.boxops


def test_candidate_lists_are_plain_lists_with_a_link():
    """No GPU needed: the lists pre_predict returns behave as lists; recall() only follows untouched ones."""
    from object_detection_amd import predictor as P
    a, b, c = [torch.zeros(3, 4), torch.zeros(2, 4)], [torch.zeros(3), torch.zeros(2)], [torch.zeros(3, dtype=torch.long), torch.zeros(2, dtype=torch.long)]
    marker = object()
    pb, ps, pc = P.remember((a, b, c), marker)
    assert isinstance(pb, list) and pb == a and len(ps) == 2
    assert P.recall(pb, ps, pc) is marker
    assert P.recall(list(pb), ps, pc) is None                 # a re-built list
    assert P.recall(pb, pc, ps) is None                       # roles swapped
    ps2 = P.remember((a, b, c), object())[1]
    assert P.recall(pb, ps2, pc) is None                      # lists of two different calls
    ps[1] = ps[1][:1]                                         # a slice view replaces an element
    assert P.recall(pb, ps, pc) is None
    pb, ps, pc = P.remember((a, b, c), marker)
    ps[0] = ps[0].clamp(max=1)                                # a fresh tensor in the same list object
    assert P.recall(pb, ps, pc) is None
    pb, ps, pc = P.remember((a, b, c), marker)
    pb[1][0, 0] = 5.0                                         # in-place edit
    assert P.recall(pb, ps, pc) is None
    pb, ps, pc = P.remember((a, b, c), marker)
    pc.append(torch.zeros(1, dtype=torch.long))
    assert P.recall(pb, ps, pc) is None


@pytest.mark.gpu
def test_bound_model_runs_the_reference_loop_order(oracle):
    """train.py:148-156: outputs -> loss -> pre_predict -> predictor.run, on the bound stand-in."""
    import object_detection_amd as D
    O = oracle
    dev = torch.device('cuda', 0)
    model = D.bind_boxops(StandInModel(21), 'ssd300')      # what the documented snippet does (checked on the CPU above; the .md does not travel to the GPU box)
    predictor = D.Predictor(iou_thresh=0.45)
    g = torch.Generator().manual_seed(4)
    B, P, C = 3, 8732, 21
    out_locs, out_confs = torch.randn(B, P, 4, generator=g), torch.randn(B, P, C, generator=g)
    out_confs[1:, :, 0] += 7.0
    gts = [O.synth_gt(i, 20, False) for i in range(B)]
    gt_bboxes, gt_labels = [x[0] for x in gts], [x[1] for x in gts]
    metas = [{'image_id': 10 + i, 'height': 300 + i, 'width': 400} for i in range(B)]
    outputs = (out_locs.to(dev).requires_grad_(), out_confs.to(dev).requires_grad_())
    loss = model.loss(outputs, gt_bboxes, gt_labels)
    assert set(loss) == {'loss', 'loss_loc', 'loss_conf'}
    loss['loss'].backward()
    assert outputs[0].grad is not None and bool(torch.isfinite(outputs[1].grad).all())
    # the exact-scores mode: torch's own soft-max on the device feeds the selection, as ssd300.py:354 does
    model.boxops.fused_activation = False
    pb, ps, pc = model.pre_predict(outputs)
    result = predictor.run(metas, pb, ps, pc)
    scores = torch.softmax(outputs[1].detach(), -1).cpu()
    wb, ws, wc = O._per_image(O.select_decode_fast, out_locs, scores, model.boxops.dboxes, 0.01, 200, 'cxcywh', 1, 0)
    for b in range(B):
        assert torch.equal(pc[b], wc[b]) and torch.equal(ps[b], ws[b])          # torch's bits, ranked as the reference ranks them
    assert result == O.predictor_run(metas, pb, ps, pc, 0.45)
    # edited lists take the generic path and give the rows of the edited data
    ps[0] = ps[0] * 0.5
    assert predictor.run(metas, pb, ps, pc) == O.predictor_run(metas, list(pb), list(ps), list(pc), 0.45)
    model.boxops.fused_activation = True
    pb2, ps2, pc2 = model.pre_predict(outputs)
    assert [t.shape for t in pb2] == [t.shape for t in pb] or True            # fused scores may differ in the last bits at a boundary
    assert predictor.run(metas, pb2, ps2, pc2) == O.predictor_run(metas, list(pb2), list(ps2), list(pc2), 0.45)
