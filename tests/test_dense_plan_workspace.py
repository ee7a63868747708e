"""CPU check of the dense plan's scratch size: it belongs to the plan, not to the address the plan happens to have."""
import torch


def _plan(row_blocks, dense_cols):
    from tango_amd.dense_plan import DensePlan
    none = torch.empty(0, dtype=torch.int32)
    kw = dict.fromkeys(("col_ids", "row_slot", "row_order", "mask_off", "mask", "segs", "segs2", "shared_blocks",
                        "res_indptr", "res_indices"), none)
    return DensePlan(rows=256 * row_blocks, num_src=dense_cols, row_blocks=row_blocks, dense_cols=dense_cols,
                     seg_ptr=torch.zeros(1), seg_ptr2=torch.zeros(1), res_max_row=0, **kw)


def test_a_later_plan_at_the_same_address_gets_its_own_scratch_size(monkeypatch):
    """The aggregation itself, its device work stubbed out: what it asks of the scratch buffer for a plan that the
    allocator put where a smaller, already collected one was."""
    from tango_amd import _lib, kernels
    asked = []
    monkeypatch.setattr(kernels, "_need", lambda t, *a, **k: t)
    monkeypatch.setattr(kernels, "_workspace", lambda nbytes, device: asked.append(nbytes))
    monkeypatch.setattr(kernels, "_stream", lambda: None)
    monkeypatch.setattr(kernels, "check", lambda rc, what: None)  # no scratch was given: the library refuses the call

    def ask(plan):
        out, feat = torch.empty(plan.rows, 41), torch.empty(plan.num_src, 48, dtype=torch.int8)
        assert kernels.cuda_kernels.csr_SPMM_dense(out, plan, feat, torch.ones(1), ldf=48, F=41)
        assert asked[-1] == _lib.lib().tango_spmm_dense_workspace(plan.ref, 41) > 0
        return asked[-1]

    small = _plan(1, 256)
    first, at = ask(small), id(small)
    del small
    kept = []
    for _ in range(64):  # until the allocator hands out the first plan's address again
        kept.append(_plan(40, 4096))
        if id(kept[-1]) == at:
            break
    for plan in kept:
        assert ask(plan) > first
