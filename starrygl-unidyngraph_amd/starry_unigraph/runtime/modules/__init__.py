from .candidates import CandidateHead
from .history import HistoryEncoder
from .time_encode import TimeEncode

__all__ = ["CandidateHead", "HistoryEncoder", "TimeEncode"]
