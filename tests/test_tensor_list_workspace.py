"""A tensor list's own workspace, without a device."""


def test_no_list_has_no_workspace():
    import aluminum_amd
    assert aluminum_amd.load().alamd_tensor_list_workspace(None) is None
