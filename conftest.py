"""Where Tila is not installed, tests of its programs are skipped with that
reason; their import would stop a session before the operators' tests, which
need no Tila, are reached."""

import pytest

NO_TILA = "Tila is not installed"


def _installed():
    try:
        import tila_b200._reference  # noqa: F401
    except ImportError:
        return False
    return True


def pytest_report_header():
    return None if _installed() else f"{NO_TILA}: tests of its programs are skipped"


@pytest.hookimpl(wrapper=True)
def pytest_make_collect_report(collector):
    report = yield
    if report.failed and isinstance(collector, pytest.Module) and "(tila-lang)" in str(report.longrepr) and not _installed():
        report.outcome = "skipped"
        report.longrepr = (str(collector.path), 1, f"Skipped: {NO_TILA}")
    return report


@pytest.hookimpl(wrapper=True)
def pytest_runtest_call(item):
    try:
        return (yield)
    except ImportError as e:
        if (e.name == "tila" or "(tila-lang)" in str(e)) and not _installed():
            pytest.skip(NO_TILA)
        raise
